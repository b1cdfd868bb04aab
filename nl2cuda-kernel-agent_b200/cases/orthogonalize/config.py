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
