"""The status word of the 8-bit operators: four bytes that the kernels may write, whatever tensor is handed over."""
import pytest
import torch

from test_int8_layouts_cpu import _last, i8  # noqa: F401  (calls are recorded instead of made)


def _calls(i8, status):  # noqa: F811
    q, one, w = torch.zeros((7, 32), dtype=torch.int8), torch.ones(7), torch.ones(32)
    return (lambda: i8.op.gemm_i8(q, one, q, one, status=status), lambda: i8.op.quantize_i8(torch.zeros((7, 32)), status=status),
            lambda: i8.op.rmsnorm_i8(torch.zeros((7, 32)), w, 1e-5, status=status))


@pytest.mark.parametrize("status", [torch.zeros(4, dtype=torch.uint8), torch.zeros(1, dtype=torch.int64), torch.zeros(1),
                                    torch.zeros(2, dtype=torch.int16), torch.zeros(0, dtype=torch.int32)],
                         ids=["bytes", "64 bits", "floating", "16 bits", "empty"])
def test_anything_but_words_is_refused(i8, status):  # noqa: F811
    for call in _calls(i8, status):
        with pytest.raises(ValueError, match="status"):
            call()
    assert not i8.calls


@pytest.mark.parametrize("dtype", [torch.int32, torch.uint32])
def test_words_are_handed_over(i8, dtype):  # noqa: F811
    status = torch.zeros(2, dtype=dtype)
    for word in (status, status[1:]):
        for call in _calls(i8, word):
            call()
            assert _last(i8).status == word.data_ptr()
