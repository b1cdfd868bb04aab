"""Shapes of the layer-norm case; LN_ROWS, LN_D and LN_DTYPE override them."""
import os

ROWS = int(os.environ.get("LN_ROWS", "4096"))
D = int(os.environ.get("LN_D", "1024"))
EPS = 1e-5
DTYPE = os.environ.get("LN_DTYPE", "float32")


def flops(rows, d):
    """Algorithmic FLOP of one forward + backward, about 8 and 12 a value."""
    return 20 * rows * d


def hbm_bytes(rows, d, elem=4):
    """Algorithmic HBM bytes of one forward + backward: x, y; then x, dy, dx."""
    return 5 * rows * d * elem
