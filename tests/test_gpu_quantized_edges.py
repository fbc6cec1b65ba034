"""8-bit pool on the GPU at the edges of what its kernels list and hold."""
import pytest

from test_gpu_quantized_shapes import check

pytestmark = pytest.mark.gpu


# ---- launches that list the most windows --------------------------------------------------------
@pytest.mark.parametrize("lead,heads,kvh,d", [(1, 8, 1, 64), (3, 2, 2, 64), (7, 16, 1, 128)])
def test_most_windows_of_a_launch(lead, heads, kvh, d):
    """Runs of 8 tokens behind `lead` tokens of another: a launch of 8192 tokens begins and ends inside
    a run, and lists 1025 windows.  Every row against the plain form."""
    runs = 2048 if lead == 1 else 1030
    spans = [(c % 37, 8) for c in range(runs)]
    check([(5, lead)] + spans, heads, kvh, d, "int8", path=7, seed=lead)
    # With two launches' ends inside runs, and runs of other lengths between them.
    mixed = [(c % 29, 8 if c % 7 else 9) for c in range(1200)]
    check([(5, lead)] + mixed, heads, kvh, d, "int8", path=7, seed=lead + 1)
