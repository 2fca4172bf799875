"""GPU: views that eas.ops gets as torch's operations make them."""

import pytest
import torch

import eas

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _ready(cuda_rt):
    yield
    cuda_rt.synchronize()
    torch.cuda.synchronize()


def test_negative_views():
    """The imaginary part of a conjugate is a view of memory that holds its negatives."""
    g = torch.Generator(device="cuda").manual_seed(0)
    w, x = torch.randn(40, 1, device="cuda", generator=g).half(), torch.randn(24, 40, device="cuda", generator=g).half()
    z = torch.view_as_complex(torch.randn(24, 1, 2, device="cuda", generator=g).half())
    part = z.conj().imag
    assert part.is_neg()
    y, want = torch.empty(24, 40, device="cuda").half(), torch.empty(24, 40, device="cuda").half()
    wx = torch.randn(8, 40, device="cuda", generator=g).half()
    for v, plain, weight in ((part, part.clone(), w), (torch._neg_view(x), -x, wx)):
        out, expect = y[:, :weight.shape[0]], want[:, :weight.shape[0]]
        eas.ops.linear(plain, weight, expect)
        for _ in range(2):    # the full path, and a repeated call
            out.fill_(7)
            eas.ops.linear(v, weight, out)
            assert torch.equal(out, expect) and expect.abs().max() > 0
    with pytest.raises(ValueError, match="negative view"):
        eas.ops.linear(x, wx, torch._neg_view(y[:, :8]))
