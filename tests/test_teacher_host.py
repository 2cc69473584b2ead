"""What the teacher's loss refuses before it launches anything: addresses of the row's weights that are no float's."""
import pytest

from annembed_amd import _lib as L

# arguments that are in order but for the row weights: the addresses are looked at, never followed
LOSS = dict(logits=4096, type=0, rows=4, cols=50, ld=50, idx=4096, list=4096, k=3, ldk=3, kind=0, temperature=1.0, weight=4096, loss=4096, stats=4096, grad=8192, ldg=50,
            work=None, work_bytes=0, stream=None)


@pytest.mark.parametrize("weight", [4097, 4098, 4099])
def test_row_weights_are_aligned(weight):
    lib = L.load()
    a = {**LOSS, "weight": weight}
    assert lib.ae_teacher_loss(*a.values()) == L.AE_ERR_INVALID_ARG
    assert "weights" in lib.ae_last_error_message().decode()
    args = [a[n] for n in ("logits", "type", "rows", "cols", "ld", "stats", "idx", "list", "k", "ldk", "kind", "temperature", "weight", "grad", "ldg", "stream")]
    assert lib.ae_teacher_grad(*args) == L.AE_ERR_INVALID_ARG
    assert "dloss" in lib.ae_last_error_message().decode()
