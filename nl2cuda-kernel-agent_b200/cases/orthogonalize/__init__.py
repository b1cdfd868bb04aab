"""Orthogonalisation case: exposes ``CASE`` for the harness."""
import os

from framework.case import Case
from cases.orthogonalize import config
from cases.orthogonalize.reference import make_inputs, reference_forward


def _description():
    with open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "description.md"),
              encoding="utf-8") as f:
        return f.read()


CASE = Case(
    name="orthogonalize",
    description=_description(),
    params={"steps": config.STEPS, "coefficients": config.COEFFICIENTS, "eps": config.EPS},
    grad_inputs=[],
    dtype=config.DTYPE,
    make_inputs=make_inputs,
    reference_forward=reference_forward,
)
