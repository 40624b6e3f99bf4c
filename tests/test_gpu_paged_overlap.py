"""Tensors that lie in one another without overlapping are taken, in place and out of it; views that overlap are refused."""
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import dev, freqs, near, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,Hq,Hkv", [(5, 8, 2), (1, 8, 2), (5, 1, 2), (5, 8, 1), (1, 1, 1), (37, 6, 3), (5, 2, 2)])
def test_in_place_beside_keys(ops, N, Hq, Hkv):  # noqa: F811
    """The output where the queries are, in one projection with keys and values; pools that are halves of one tensor, page by page and head by head."""
    D, page, pages = 64, 4, 12
    for interleaved in (False, True):
        qkv = torch.randn(N, Hq + 2 * Hkv, D, device="cuda").half()
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        both = torch.zeros(pages, page, Hkv, 2, D, device="cuda").half() if interleaved else torch.zeros(pages, 2, page, Hkv, D, device="cuda").half()
        kp, vp = (both[:, :, :, i] for i in range(2)) if interleaved else (both[:, i] for i in range(2))
        pos, f, slots = dev(list(range(3, 3 + N))), freqs(D // 2), dev(list(range(N)))
        want, before = plain.rotate(qkv.cpu(), pos.cpu(), f, "half"), qkv.clone()
        bound = plain.rotate_bound(qkv.cpu(), want, f, "half", 1.0)
        assert ops.rotary_paged_store(q, k, v, pos, slots, f.cuda(), kp, vp, out=q) is q
        near(q, want[:, :Hq], bound[:, :Hq])
        assert torch.equal(qkv[:, Hq:], before[:, Hq:])
        rows, cols = torch.arange(N).cuda() // page, torch.arange(N).cuda() % page
        near(kp[rows, cols], want[:, Hq:Hq + Hkv], bound[:, Hq:Hq + Hkv])
        assert torch.equal(vp[rows, cols], v)
        spare = torch.zeros(N, 2 * Hq + 1, D, device="cuda").half()
        spare[:, :Hq] = before[:, :Hq]
        ops.rotary(spare[:, :Hq], pos, f.cuda(), out=spare[:, Hq + 1:])
        near(spare[:, Hq + 1:], want[:, :Hq], bound[:, :Hq])
        assert torch.equal(spare[:, :Hq], before[:, :Hq]) and not bool(spare[:, Hq].any())
        table, lengths = dev([[0, 1]] * N), dev([min(n + 1, 2 * page) for n in range(N)])
        if Hq % Hkv == 0:
            want, _, bound, _ = plain.attend(before[:, :Hq], kp, vp, table, lengths.tolist(), 0.3)
            ops.paged_attn(before[:, :Hq], kp, vp, table, lengths, 0.3, out=spare[:, Hq + 1:])
            near(spare[:, Hq + 1:], want, bound)
            ops.paged_attn(before[:, :Hq], kp, vp, table, lengths, 0.3, out=before[:, :Hq])
            assert torch.equal(before[:, :Hq], spare[:, Hq + 1:])


def test_views_that_overlap(ops):  # noqa: F811
    from kvcomp_b200._lib import KvcError
    x, pos, f = torch.randn(9, 4, 64, device="cuda").half(), dev(list(range(8))), freqs(32).cuda()
    whole = torch.zeros(40, 4, 64, device="cuda").half()
    pool, slots = torch.zeros(6, 4, 4, 64, device="cuda").half(), dev(list(range(8)))
    before = x.clone()
    for out in (x[1:], x[:1].expand(8, 4, 64), whole[:8, :1].expand(8, 4, 64), whole.view(-1)[:8 * 64].view(8, 1, 64).expand(8, 4, 64), x.view(-1)[64:64 + 8 * 256].view(8, 4, 64)):
        with pytest.raises(KvcError, match="overlap"):
            ops.rotary(x[:8], pos, f, out=out)
        with pytest.raises(KvcError, match="overlap"):
            ops.paged_attn(x[:8], pool, pool, dev([[0]] * 8), dev([1] * 8), 0.1, out=out)
    k = whole[:8]
    for kp, vp in ((pool[:1].expand(6, 4, 4, 64), pool.clone()), (pool, pool[:, :, :1].expand(6, 4, 4, 64)), (pool[:5], pool[1:]), (pool, pool)):
        with pytest.raises(KvcError, match="overlap"):
            ops.rotary_paged_store(None, k, k, pos, slots, f, kp, vp)
    with pytest.raises(KvcError, match="overlap"):
        ops.rotary_paged_store(x[:8], k, whole[8:16], pos, slots, f, pool, pool.clone(), out=whole[4:12])
    assert torch.equal(x, before) and not bool(whole.any()) and not bool(pool.any())
