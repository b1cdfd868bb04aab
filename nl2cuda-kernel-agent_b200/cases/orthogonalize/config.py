"""Shapes of the orthogonalisation case; ORTHO_M, ORTHO_N and ORTHO_DTYPE override them."""
import os

M = int(os.environ.get("ORTHO_M", "1024"))
N = int(os.environ.get("ORTHO_N", "2048"))
STEPS = 5
# Each step maps a singular value s to a s + b s^3 + c s^5: five steps of these bring every one
# above about 1/500 of the Frobenius norm near 1 (0.7 to 1.2).
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
DTYPE = os.environ.get("ORTHO_DTYPE", "float32")


def flops(m, n, steps=STEPS):
    """Algorithmic FLOP: a step's X X^T and A^2 (symmetric: half of each) and B X."""
    r, c = min(m, n), max(m, n)
    return steps * (3 * r * r * c + r ** 3)


def hbm_bytes(m, n, elem=4):
    """Bytes that cannot be avoided: the update read, the result written."""
    return 2 * m * n * elem
