"""Shapes of the layer-norm case; LN_ROWS, LN_D and LN_DTYPE override them."""
import os

ROWS = int(os.environ.get("LN_ROWS", "4096"))
D = int(os.environ.get("LN_D", "1024"))
EPS = 1e-5
DTYPE = os.environ.get("LN_DTYPE", "float32")
