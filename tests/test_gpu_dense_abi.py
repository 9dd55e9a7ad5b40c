"""wf_dense at the ends of its arguments' ranges."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("rows_per_group", [1 << 20, 1 << 32, (1 << 32) + 1, 1 << 62])
def test_a_group_longer_than_the_rows(native, rows, rows_per_group):
    # one gate row for all, as with rows_per_group = rows (in the few-rows form and in tiles)
    fd = sub("enhancers.fused_dense")
    x, w = (torch.randn(n, 128, device="cuda").to(torch.bfloat16) for n in (rows, 64))
    gate = torch.randn(64, device="cuda").to(torch.bfloat16)
    want, y = fd.dense(x, w, gate=gate), torch.empty(rows, 64, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    rc = native.lib().wf_dense(x.data_ptr(), 128, 1, w.data_ptr(), 128, 1, 1, rows, 64, 128, None, 1, 0, gate.data_ptr(), 1,
                               rows_per_group, None, 0, y.data_ptr(), None, ws.data_ptr(), ws.numel(),
                               native.stream_of(x.device))
    assert rc == native.OK and torch.equal(y, want)
