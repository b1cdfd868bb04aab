"""CTA pairs that end at once: the leader's last commits arrive in both CTAs, and each waits for its own.

Calls of one tile, whose CTAs have next to nothing to do between their first MMA and their exit, back to
back: every result is the first one's, and no wait runs out.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 1), (8, 64), (40, 70), (2, 16, 200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_update_of_one_tile(shape, dtype, cuda_device, monkeypatch):
    from cases.orthogonalize.op import orthogonalize
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    g = torch.randn(shape, device="cuda", generator=gen).to(dtype)
    for steps in (1, 5):
        want = orthogonalize(g, steps)
        outs = [orthogonalize(g, steps) for _ in range(100)]
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)
    monkeypatch.setenv("RBF_CHECK_STATUS", "1")
    assert torch.equal(orthogonalize(g, steps), want)


@pytest.mark.parametrize("n,m,d", [(4, 4, 4), (100, 128, 32), (256, 128, 64), (600, 260, 64)])
def test_pairwise_forward_of_few_tiles(n, m, d, cuda_device, monkeypatch):
    from cases.rbf import native
    monkeypatch.setenv("RBF_FWD_PAIR", "1")
    gen = torch.Generator(device="cuda").manual_seed(n + m + d)
    x, y = (torch.randn(r, d, device="cuda", generator=gen) for r in (n, m))
    want = native.rbf_forward(x, y, 0.1)
    outs = [native.rbf_forward(x, y, 0.1) for _ in range(100)]
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)
