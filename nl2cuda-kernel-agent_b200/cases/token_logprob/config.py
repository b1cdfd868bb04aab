"""Shapes of the token log-probability case; LP_B, LP_T, LP_V and LP_DTYPE override them."""
import os

B = int(os.environ.get("LP_B", "8"))      # sequences
T = int(os.environ.get("LP_T", "64"))     # positions of each
V = int(os.environ.get("LP_V", "8192"))   # vocabulary
IGNORE_INDEX = -100
DTYPE = os.environ.get("LP_DTYPE", "float32")
