"""What happens when a bounded wait of the attention kernel runs out: the call returns, the status word says so, and the device
works on."""
import pytest
import torch

from test_gpu_attention import cu, dev, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (128, "fp16"), (256, "bf16")])
@pytest.mark.parametrize("lens", [(3000, 700), (40,)])
def test_waits_that_may_not_last(monkeypatch, lens, d, dtype):
    """No wait may last: where one has to, the kernel winds down (with loads, products and arrivals of both CTAs of a pair under
    way) and says so; where none has to, the answer is right. The next calls are as if nothing had been."""
    import reax_engine_b200 as R
    from reax_engine_b200 import _lib as L
    c = dev(cu(lens))
    q, k, v, pk, pv = tensors(sum(lens), sum(lens), 16, 8, d, dtype, d, prefix=500)
    want = R.shared_prefix_attention(q, k, v, pk, pv, c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        monkeypatch.setenv("REAXMOE_WAIT_TIMEOUT_NS", "0")
        got = R.shared_prefix_attention(q, k, v, pk, pv, c, status=status)
        monkeypatch.delenv("REAXMOE_WAIT_TIMEOUT_NS")
        code = int(status)
        assert code in (0, L.ERR_DEVICE_TIMEOUT)
        if len(lens) > 1:
            assert code == L.ERR_DEVICE_TIMEOUT
        if code == 0:
            assert torch.equal(got, want)
        status.zero_()
        assert torch.equal(R.shared_prefix_attention(q, k, v, pk, pv, c, status=status), want) and int(status) == 0
