"""Shapes of the policy-loss case; POLICY_B, POLICY_T, POLICY_V and POLICY_DTYPE override them."""
import os

B = int(os.environ.get("POLICY_B", "8"))      # sequences
T = int(os.environ.get("POLICY_T", "64"))     # positions of each
V = int(os.environ.get("POLICY_V", "8192"))   # vocabulary
IGNORE_INDEX = -100
CLIP_LOW = 0.2
CLIP_HIGH = 0.2
KL_COEF = 0.05
DTYPE = os.environ.get("POLICY_DTYPE", "float32")
