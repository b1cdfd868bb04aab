"""Policy-loss case: exposes ``CASE`` for the harness."""
import os

from framework.case import Case
from cases.policy_loss import config
from cases.policy_loss.reference import make_inputs, reference_forward


def _description():
    with open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "description.md"),
              encoding="utf-8") as f:
        return f.read()


CASE = Case(
    name="policy_loss",
    description=_description(),
    params={"clip_low": config.CLIP_LOW, "clip_high": config.CLIP_HIGH,
            "kl_coef": config.KL_COEF, "ignore_index": config.IGNORE_INDEX},
    grad_inputs=["logits"],
    dtype=config.DTYPE,
    make_inputs=make_inputs,
    reference_forward=reference_forward,
)
