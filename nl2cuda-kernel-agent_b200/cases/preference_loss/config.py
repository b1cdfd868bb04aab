"""Shapes of the preference-loss case; PREF_B, PREF_T, PREF_V and PREF_DTYPE override them."""
import os

B = int(os.environ.get("PREF_B", "8"))      # sequences
T = int(os.environ.get("PREF_T", "64"))     # positions of each
V = int(os.environ.get("PREF_V", "8192"))   # vocabulary
IGNORE_INDEX = -100
BETA = 0.1
LABEL_SMOOTHING = 0.0
DTYPE = os.environ.get("PREF_DTYPE", "float32")
