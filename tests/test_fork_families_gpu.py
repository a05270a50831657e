"""Forks of models that keep state, pooled blocks, windows or latents (`fork_families.py`).  Tolerance: that of the families' own replays in
float32, sums in another order than the plain implementation's."""
import pytest

from fork_families import CASES, check_forks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("family,name", CASES)
def test_forks(family, name, graphs):
    check_forks(family, name, (32, 77) if graphs else (9,), 3e-5, dtype="float32", use_graphs=graphs)
