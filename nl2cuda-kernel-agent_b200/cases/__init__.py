"""Algorithm cases: the pairwise matrices (``rbf``, ``cosine_sim``) and the operators of a
language-model fine-tuning step (``layernorm``, ``token_logprob``, ``preference_loss``,
``policy_loss``, ``orthogonalize``)."""
