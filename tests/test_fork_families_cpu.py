"""Forks of models that keep state, pooled blocks, windows or latents, with plain kernels (`fork_families.py`).  Tolerance: that of the families'
own tests on the CPU, float32 sums in another order than the plain implementation's."""
import pytest

from draft_ops import PlainTreeOps
from fork_families import CASES, check_forks


@pytest.mark.parametrize("family,name", CASES)
def test_forks(family, name):
    check_forks(family, name, (9, 32), 3e-5, dtype="float32", device="cpu", ops=PlainTreeOps())
