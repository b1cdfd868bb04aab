"""Layer-norm case: exposes ``CASE`` for the harness."""
import os

from framework.case import Case
from cases.layernorm import config
from cases.layernorm.reference import make_inputs, reference_forward


def _description():
    with open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "description.md"),
              encoding="utf-8") as f:
        return f.read()


CASE = Case(
    name="layernorm",
    description=_description(),
    params={"eps": config.EPS},
    grad_inputs=["x", "weight", "bias"],
    dtype=config.DTYPE,
    make_inputs=make_inputs,
    reference_forward=reference_forward,
)
