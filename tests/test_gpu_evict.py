"""Eviction of packed groups and of full-precision tokens by weight: selections against plain sorting, bytes against indexing."""

import math

import pytest
import torch

import chunk_reference as ref

pytestmark = pytest.mark.gpu


def packs(B, H, T, bits, dtype=torch.float16, seed=0):
    g = torch.Generator().manual_seed(seed)
    word = lambda *s: torch.randint(-2 ** 31, 2 ** 31, s, generator=g).to(torch.int32).cuda()
    num = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    return (word(B, H, 128, T * bits // 32), num(B, H, 128, T // 32), num(B, H, 128, T // 32)), \
        (word(B, H, T, 4 * bits), num(B, H, T, 4), num(B, H, T, 4))


def weights(kind, B, H, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(3 * torch.randn(B, H, n, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, (B, H, n), generator=g).float()
    elif kind == "equal":
        w = torch.full((B, H, n), 0.25)
    elif kind == "special":
        w[..., ::7], w[..., 3::11], w[..., 5::13], w[..., 1::5] = math.inf, math.nan, -math.inf, 0.0
        w[..., 2::5] = -0.0
        w[..., 4::17] = -1e-40
    elif kind == "near":      # sums that differ in the last bits of 32 numbers
        w = 1 + torch.randint(0, 2, (B, H, n), generator=g) * 2.0 ** -23
    return w


def gather_groups(t, kept, dim, per):
    """Blocks of ``per`` along ``dim`` (2 or 3) of t [B,H,..]."""
    idx = (kept[..., None] * per + torch.arange(per)).flatten(2)
    idx = idx[..., None].expand(-1, -1, -1, t.shape[3]) if dim == 2 else idx[:, :, None].expand(-1, -1, t.shape[2], -1)
    return t.cpu().gather(dim, idx)


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "special", "near"])
@pytest.mark.parametrize("B,H,T,keep,bits", [(1, 1, 32, 1, 4), (2, 2, 320, 3, 4), (1, 3, 1280, 40, 2), (2, 1, 4128, 64, 1), (1, 2, 33 * 32, 32, 4),
                                             (1, 1, 640 * 32, 333, 4)])
def test_groups(B, H, T, keep, bits, kind):
    from calibquant_b200 import ops
    kp, vp = packs(B, H, T, bits, torch.bfloat16 if bits == 2 else torch.float16, seed=T)
    w = weights(kind, B, H, T, seed=keep)
    k2, v2, w2, kept = ops.evict_groups(kp, vp, w.cuda(), keep, bits=bits)
    total = w.double().unflatten(-1, (-1, 32)).sum(-1)
    want = ref.kept_largest(total, keep)
    assert kept.dtype == torch.int64 and torch.equal(kept.cpu(), want)
    for got, t, per in zip(k2, kp, (bits, 1, 1)):
        assert got.dtype == t.dtype and torch.equal(got.cpu(), gather_groups(t, want, 3, per))
    for got, t in zip(v2, vp):
        assert got.dtype == t.dtype and torch.equal(got.cpu(), gather_groups(t, want, 2, 32))
    assert torch.equal(w2.cpu().view(torch.int32), gather_groups(w[..., None], want, 2, 32)[..., 0].view(torch.int32))


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "special"])
@pytest.mark.parametrize("B,H,t_fp,keep,sys,recent,cap", [(1, 1, 1, 1, 0, 0, 1), (1, 2, 300, 160, 41, 32, 300), (2, 2, 77, 60, 41, 19, 128), (2, 1, 513, 513, 41, 5, 600),
                                                          (1, 3, 1025, 7, 0, 0, 1100), (1, 1, 9000, 4001, 41, 256, 9000), (2, 2, 50, 20, 20, 0, 50)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tokens(B, H, t_fp, keep, sys, recent, cap, kind, dtype):
    from calibquant_b200 import ops
    g = torch.Generator().manual_seed(cap)
    k, v = (torch.randn(B, H, cap, 128, generator=g).to(dtype) for _ in range(2))
    w = weights(kind, B, H, cap, seed=keep)
    k2, v2, w2, kept = ops.evict_tokens(k.cuda(), v.cuda(), w.cuda(), keep, t_sys=sys, recent=recent, t_fp=t_fp)
    rest = ref.kept_largest(w[..., sys:t_fp - recent], keep - sys - recent) + sys if keep > sys + recent else torch.empty(B, H, 0, dtype=torch.int64)
    ends = lambda r: torch.tensor(list(r), dtype=torch.int64).expand(B, H, -1)
    want = torch.cat([ends(range(sys)), rest, ends(range(t_fp - recent, t_fp))], -1)
    assert torch.equal(kept.cpu(), want)
    row = want[..., None].expand(-1, -1, -1, 128)
    assert torch.equal(k2.cpu(), k.gather(2, row)) and torch.equal(v2.cpu(), v.gather(2, row))
    assert torch.equal(w2.cpu().view(torch.int32), w.gather(2, want).view(torch.int32))


def test_layouts():
    """Strided caches and weights, tensors that start off a 16-byte boundary."""
    from calibquant_b200 import ops
    k, v = (torch.randn(2, 60, 3, 128, device="cuda").half().transpose(1, 2) for _ in range(2))
    w = torch.rand(2, 3, 80, device="cuda")
    a = ops.evict_tokens(k, v, w[..., 7:67], 30, 10, 5)
    b = ops.evict_tokens(k.contiguous(), v.contiguous(), w[..., 7:67].contiguous(), 30, 10, 5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    kp, vp = packs(1, 2, 320, 4)
    off = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)
    w = torch.rand(1, 2, 320, device="cuda")
    a, b = ops.evict_groups(kp, vp, w, 4), ops.evict_groups([off(t) for t in kp], [off(t) for t in vp], off(w), 4)
    assert all(torch.equal(x, y) for x, y in zip((*a[0], *a[1], *a[2:]), (*b[0], *b[1], *b[2:])))


def test_refusals():
    from calibquant_b200 import ops
    kp, vp = packs(1, 2, 64, 4)
    w = torch.rand(1, 2, 64, device="cuda")
    for args in ((kp, vp, w, 0), (kp, vp, w, 3), (kp, vp, w[..., :32], 1), (kp, kp, w, 1), (kp, vp, w.half(), 1), (kp, vp, w, 1, 2), (kp, vp, w, 1, 8),
                 (kp, vp, w, 1, 4, 64), (kp[:2], vp, w, 1), (None, vp, w, 1)):
        with pytest.raises((ValueError, TypeError)):
            ops.evict_groups(*args)
    with pytest.raises(RuntimeError):
        ops.evict_groups(kp, vp, w.cpu(), 1)
    k = torch.randn(1, 2, 64, 128, device="cuda").half()
    for kw in (dict(keep=0), dict(keep=65), dict(keep=40, t_fp=39), dict(keep=10, t_sys=11), dict(keep=10, t_sys=5, recent=6), dict(keep=10, t_sys=-1),
               dict(keep=10, t_fp=70), dict(keep=10, weights=w[..., :63]), dict(keep=10, v_fp=k[:, :1]), dict(keep=10, k_fp=k.float()),
               dict(keep=10, weights=w[0])):
        with pytest.raises((ValueError, TypeError)):
            ops.evict_tokens(**{**dict(k_fp=k, v_fp=k, weights=w), **kw})
    big = torch.empty(1, 1, 24577, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        ops.evict_tokens(big, big, torch.zeros(1, 1, 24577, device="cuda"), 5)


def test_results_are_tensors_of_their_own():
    """Results that share an allocation neither overlap nor know of one another: in-place changes, views, autograd's version counters, copies."""
    from calibquant_b200 import ops
    k = torch.randn(2, 2, 40, 128, device="cuda").half()
    w = torch.rand(2, 2, 40, device="cuda")
    k2, v2, w2, kept = ops.evict_tokens(k, -k, w, 7)
    kp, vp = ops.pack_k_per_channel(k[:, :, :32].contiguous(), 32, 4), ops.pack_v_per_token(k[:, :, :32].contiguous(), 32, 4)
    groups = ops.evict_groups(kp, vp, w[:, :, :32].contiguous(), 1)
    for results in ((k2, v2, w2, kept), (*groups[0], *groups[1], *groups[2:])):
        before = [t.clone() for t in results]
        for i, t in enumerate(results):
            versions = [u._version for u in results]
            assert t.is_contiguous() and t.data_ptr() % 256 == 0 and t.device == k.device
            t.zero_()
            assert [u._version for u in results] == [v + (j == i) for j, v in enumerate(versions)]
            assert all(torch.equal(u, b) for u, b in zip(results[i + 1:], before[i + 1:])) and not t.any()
    x = torch.zeros_like(w2).requires_grad_()
    (x * w2).sum().backward()
    assert x.grad.shape == w2.shape
