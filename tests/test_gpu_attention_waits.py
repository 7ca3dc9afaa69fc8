"""What happens when a bounded wait of the attention kernel runs out: the call returns, the status word says so, and the device
works on."""
import pytest
import torch

from test_gpu_attention import check, cu, dev, reference, tensors

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


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_done_key_by_key_do_not_run_out_the_waits_for_them(monkeypatch, d):
    """One pair of CTAs, several items, and in each a last key whose value is NaN, which only the last row sees: the other rows of
    its tile are done again one key after another, which takes far longer than the waits may last without a sign of life."""
    import reax_engine_b200 as R
    m, n, h = 128, 12000, 4
    q, k, v, _, _ = tensors(m, n, h, h, d, "bf16", d)
    v[-1] = float("nan")
    c, ck = dev([0, m]), dev([0, n])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 9.0)
    try:
        R.set_sm_budget(2)
        monkeypatch.setenv("REAXMOE_WAIT_TIMEOUT_NS", "5000000")
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        _, lse = R.prompt_attention(q, k, v, c, ck, out=out, status=status, return_lse=True)
        end.record()
        torch.cuda.synchronize()
    finally:
        R.set_sm_budget(0)
    assert int(status) == 0
    assert start.elapsed_time(end) > 50          # ms: ten times the limit
    assert torch.isnan(out[-1].float()).all()
    rows = [0, 63, 126]
    for r in rows:
        ref = reference(q[r:r + 1], k[:n - m + r + 1], v[:n - m + r + 1], [0, 1], [0, n - m + r + 1], d ** -0.5)
        check(out[r:r + 1], ref, lse[r:r + 1])


def test_a_call_without_a_status_word_is_reported(monkeypatch):
    import reax_engine_b200 as R
    from reax_engine_b200 import _lib as L
    c = dev([0, 3000])
    q, k, v, _, _ = tensors(3000, 3000, 8, 4, 128, "bf16", 1)
    want = R.prompt_attention(q, k, v, c)
    assert R.attention_status() == 0
    monkeypatch.setenv("REAXMOE_WAIT_TIMEOUT_NS", "0")
    R.prompt_attention(q, k, v, c)
    monkeypatch.delenv("REAXMOE_WAIT_TIMEOUT_NS")
    assert R.attention_status("cuda:0", clear=False) == L.ERR_DEVICE_TIMEOUT
    assert R.attention_status(0) == L.ERR_DEVICE_TIMEOUT and R.attention_status(torch.device("cuda")) == 0
    assert torch.equal(R.prompt_attention(q, k, v, c), want) and R.attention_status() == 0
