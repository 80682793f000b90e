"""Chunk attention and key weights where a tile, a row or a whole block of rows has next to nothing to look at."""

import math

import pytest
import torch

import chunk_reference as ref
from test_gpu_chunk import BF16, HALF, check, make

pytestmark = pytest.mark.gpu


def lowest_rows(out, v, first, n):
    """Query i of the first n sees keys ``first`` .. i, all at bfloat16's lowest value: every key counts alike, exactly (the mask's step in fp32 is 2^104,
    so that scores drown in it; fp16's lowest value has one of 2^-8, and they do not), and the output is a plain mean of values.  Its sum is cut off at 2^-22 of its largest term per 16 keys, then rounded once."""
    for i in range(n):
        rows = v[:, :, first:i + 1].cpu().double()
        rep = out.shape[2] // rows.shape[1]
        want = rows.mean(2).repeat_interleave(rep, 1)
        room = torch.finfo(out.dtype).eps / 2 * want.abs() + 2.0 ** -18 * rows.abs().mean(2).repeat_interleave(rep, 1) + torch.finfo(out.dtype).tiny
        assert ref.within(out[:, i], want, room), i


@pytest.mark.parametrize("dtype", [HALF, BF16])
@pytest.mark.parametrize("shape,masked", [
    ((16, 32, 8, 20, 0, 246), (0, 246)),          # the even half of the key tiles: one that is masked as a whole, one that ten queries do not see
    ((6, 16, 4, 28, 1152, 370), (96, 370)),       # behind a visual span, five parts
    ((40, 8, 4, 33, 1056, 300), (41, 300)),       # a part per half, six key tiles each
    ((16, 8, 8, 300, 0, 0), (0, 10)),             # left padding: the first queries see nothing but the padding, then a tile they do not see
    ((16, 8, 8, 300, 0, 129), (0, 129)),
    ((4, 24, 8, 430, 0, 0), (0, 120)),            # the same with key tiles unpacked once
], ids=str)
def test_lowest_masks_in_front_of_hidden_tiles(shape, masked, dtype):
    """Padding at the type's lowest value (not -inf) in one tile, and a tile without a mask behind it that causality hides."""
    B, Hq, Hkv, L, t_vis, before = shape
    q, kp, vp, k_fp, v_fp = make(*shape, dtype, seed=L)
    t_sys = min(41, before)
    mask = torch.zeros(B, t_vis + before + L, dtype=dtype, device="cuda")
    order = torch.cat([torch.arange(t_sys), torch.arange(t_sys + t_vis, t_vis + before + L)])      # places of the full-precision tokens
    mask[:, order[masked[0]:masked[1]].cuda()] = torch.finfo(dtype).min
    out, lse, w = check(q, kp, vp, k_fp, v_fp, t_sys, mask)
    if dtype == BF16 and t_vis == 0 and before == 0:
        lowest_rows(out, v_fp, 0, masked[1])


@pytest.mark.parametrize("dtype", [HALF, BF16])
def test_lowest_masks_over_everything_old(dtype):
    """The visual span and the text before the new tokens at the lowest value, the new tokens' own first ones as well."""
    q, kp, vp, k_fp, v_fp = make(16, 8, 8, 300, 64, 20, dtype, seed=2)
    mask = torch.zeros(16, 384, dtype=dtype, device="cuda")
    mask[::2, :84 + 30] = torch.finfo(dtype).min
    mask[1::2, :84] = -math.inf
    mask[1::2, 84:84 + 30] = torch.finfo(dtype).min
    out, lse, _ = check(q, kp, vp, k_fp, v_fp, 20, mask)
    if dtype == BF16:
        lowest_rows(out[1::2], v_fp[1::2, :, 20:], 0, 30)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("shape", [(2, 8, 2, 1, 64, 20), (2, 8, 2, 40, 192, 20), (16, 8, 8, 300, 64, 20), (4, 24, 8, 430, 0, 9)], ids=str)
def test_a_query_that_is_not_a_number(shape, masked):
    """Its row is NaN in all three results, whatever way the partial results take (few rows, merged parts, one part, images); the others are what they were."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(*shape, BF16, seed=9)
    B, Hq, Hkv, L = shape[:4]
    mask = torch.randn(B, shape[4] + k_fp.shape[2], device="cuda").bfloat16() if masked else None
    want = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 9, mask=mask, return_lse=True)
    q[1, L // 2, 3, 5] = math.nan
    got = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 9, mask=mask, return_lse=True)
    assert torch.isnan(got[0][1, L // 2, 3]).all() and torch.isnan(got[1][1, 3, L // 2])
    w = ops.key_weights(q, got[1], kp, k_fp, 9, mask=mask)
    seen = k_fp.shape[2] - L + L // 2 + 1
    assert torch.isnan(w[0][1, 3 // (Hq // Hkv)]).all() and torch.isnan(w[1][1, 3 // (Hq // Hkv), :seen]).all()
    got[0][1, L // 2, 3], got[1][1, 3, L // 2] = want[0][1, L // 2, 3], want[1][1, 3, L // 2]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [HALF, BF16])
@pytest.mark.parametrize("shape", [(16, 8, 8, 300, 0, 0), (4, 24, 8, 430, 0, 0)], ids=str)
def test_row_blocks_without_a_key(shape, dtype):
    """Fewer live tokens than new ones and no visual span: whole row blocks of one part see nothing, and give zeros, whatever the queries are."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(*shape, dtype, seed=7)
    t_fp = k_fp.shape[2]
    for live in (20, 1, 0):
        k_fp[:, :, live:], v_fp[:, :, live:] = math.nan, math.nan
        counter = torch.tensor([live], dtype=torch.int32, device="cuda")
        out, lse, w = check(q, kp, vp, k_fp, v_fp, 0, t_fp=t_fp, t_fp_dev=counter, live=live)
        none = shape[3] - live
        assert not out[:, :none].any() and torch.isneginf(lse[..., :none]).all()
        for _ in range(20):
            again = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 0, t_fp=t_fp, t_fp_dev=counter, return_lse=True)
            assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def sized(B, Hq, Hkv, L, t_vis, before, dtype, key, query, seed=0):
    """Inputs whose keys are of size ``key`` (channels lognormal about it) and queries of size ``query``."""
    from calibquant_b200 import ops
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    f = torch.exp(rnd(128)) * key
    kp = ops.pack_k_per_channel((rnd(B, Hkv, t_vis, 128) * f).to(dtype).cuda(), 32, 4)
    vp = ops.pack_v_per_token(rnd(B, Hkv, t_vis, 128).to(dtype).cuda(), 32, 4)
    fp = lambda s: (rnd(B, Hkv, before + L, 128) * s).to(dtype).cuda()
    return (rnd(B, L, Hq, 128) * query).to(dtype).cuda(), kp, vp, fp(f), fp(1.0)


@pytest.mark.parametrize("key,query", [(1e-2, 30.0), (1e-3, 300.0), (2e-4, 1500.0), (300.0, 1e-3), (2e-4, 1.0), (300.0, 1e-2)])
@pytest.mark.parametrize("L", [1, 4])
def test_small_keys_and_large_queries_of_few_rows(L, key, query):
    """fp16 far from one: the product of a query and a scale in two terms keeps 22 bits wherever in the range they lie."""
    q, kp, vp, k_fp, v_fp = sized(2, 8, 2, L, 256, 20, HALF, key, query, seed=L)
    check(q, kp, vp, k_fp, v_fp, 20)
    q[..., ::3] *= 2.0 ** -9                             # channels far below the row's largest
    check(q, kp, vp, k_fp, v_fp, 20)


def test_ends_of_fp16_of_few_rows():
    """Scales from subnormal to the largest number beside one another, queries at either end."""
    q, kp, vp, k_fp, v_fp = sized(1, 8, 2, 2, 128, 20, HALF, 1.0, 1.0)
    for g, s in enumerate((6e-8, 6.2e-5, 1.0, 65504.0)):
        kp[1][..., g] = s * torch.randint(1, 2, (1, 2, 128), device="cuda")
        kp[2][..., g] = 0
    q[:] = 0
    q[..., 5], q[..., 9] = 6e-8, -6e-8                   # scores of 65504 * 15 * 2^-24 at most
    check(q, kp, vp, k_fp, v_fp, 20)
    kp[1][..., 2:] = 0
    q[..., 5], q[..., 9] = 60000.0, 2.0                  # of 6e4 * 15 * 2^-14
    check(q, kp, vp, k_fp * 1e-5, v_fp, 20)


@pytest.mark.parametrize("key,query", [(1e-2, 30.0), (1e-3, 300.0), (2e-4, 1500.0), (300.0, 1e-3), (2e-4, 1.0), (300.0, 1e-2)])
@pytest.mark.parametrize("L", [24, 390])
def test_small_keys_and_large_queries(L, key, query):
    """The same for the tiles of the tensor core, with key tiles unpacked in the kernel and once before it."""
    q, kp, vp, k_fp, v_fp = sized(1, 8, 2, L, 256, 20, HALF, key, query, seed=L)
    check(q, kp, vp, k_fp, v_fp, 20)
