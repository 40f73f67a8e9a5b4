"""Every launch of an 8-bit step that waits for copies reports to the model's status word."""
import pytest

from test_step_int8_cpu import model  # noqa: F401  (the recorders)


@pytest.mark.parametrize("logits", [False, True])
def test_rows_and_products_report_to_the_models_word(model, logits):  # noqa: F811
    m, calls = model
    m._launch_step(0, logits)
    kernels = [k for name, _, k in calls if name in ("rmsnorm_i8", "quantize_i8", "gemm_i8")]
    assert len(kernels) == 2 * 8 + 2 * logits and all(k["status"] is m.status for k in kernels)
