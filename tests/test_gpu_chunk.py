"""Attention of several new tokens on a 4-bit cache, and the weights of its keys, against 64-bit forms."""

import math

import pytest
import torch

import chunk_reference as ref

pytestmark = pytest.mark.gpu
HALF, BF16 = torch.float16, torch.bfloat16


def make(B, Hq, Hkv, L, t_vis, before, dtype, seed=0, offset=0.0, cap=None):
    """q, packs, full-precision cache of 41 + before + L tokens (room for ``cap``) on the GPU."""
    from calibquant_b200 import ops
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    f = torch.exp(rnd(128)) * 0.7
    bias = offset * rnd(128)
    t_fp = before + L
    kp = vp = None
    if t_vis:
        kp = ops.pack_k_per_channel(((rnd(B, Hkv, t_vis, 128) + bias) * f).to(dtype).cuda(), 32, 4)
        vp = ops.pack_v_per_token(rnd(B, Hkv, t_vis, 128).to(dtype).cuda(), 32, 4)
    k_fp = ((rnd(B, Hkv, cap or t_fp, 128) + bias) * f).to(dtype).cuda()
    v_fp = rnd(B, Hkv, cap or t_fp, 128).to(dtype).cuda()
    q = rnd(B, L, Hq, 128).to(dtype).cuda()
    return q, kp, vp, k_fp, v_fp


def check(q, kp, vp, k_fp, v_fp, t_sys, mask=None, t_fp=None, t_fp_dev=None, live=None):
    """Attention, log-sum-exp and weights of one set of inputs."""
    from calibquant_b200 import ops
    kw = dict(mask=mask, t_fp=t_fp, t_fp_dev=t_fp_dev)
    out, lse = ops.chunk_attention(q, kp, vp, k_fp, v_fp, t_sys, return_lse=True, **kw)
    n = t_fp if t_fp is not None else k_fp.shape[2]
    args = (q, kp, k_fp[:, :, :n], t_sys, mask, live)
    want_o, want_l, room_o, room_l = ref.attention64(q, kp, vp, k_fp[:, :, :n], v_fp[:, :, :n], t_sys, mask, live)
    assert ref.within(lse, want_l, room_l)
    assert ref.within(out, want_o, room_o)
    w = ops.key_weights(q, lse, kp, k_fp, t_sys, **kw)
    want_w, room_w = ref.weights64(q, lse, *args[1:])
    assert w[0].shape == want_w[0].shape and w[1].shape == want_w[1].shape
    assert ref.within(w[0], want_w[0], room_w[0]) and ref.within(w[1], want_w[1], room_w[1])
    assert ops.device_status() == 0
    return out, lse, w


SHAPES = [      # B, Hq, Hkv, L, T_vis, tokens before
    (1, 4, 1, 1, 32, 0), (1, 8, 2, 1, 256, 64), (2, 8, 2, 3, 96, 41), (1, 2, 2, 1, 0, 5), (1, 4, 4, 130, 0, 0), (3, 12, 2, 7, 160, 130),
    (1, 8, 1, 16, 128, 1), (1, 8, 1, 17, 384, 127), (1, 6, 1, 43, 64, 44), (2, 4, 1, 65, 32, 300), (1, 16, 2, 129, 416, 87),
    (1, 32, 8, 5, 1312, 41), (1, 10, 1, 13, 224, 9), (1, 2, 1, 513, 96, 3), (1, 1, 1, 1, 4128, 0), (2, 8, 8, 64, 64, 64), (1, 48, 8, 3, 640, 50),
]


@pytest.mark.parametrize("dtype", [HALF, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, dtype):
    q, kp, vp, k_fp, v_fp = make(*shape, dtype, seed=sum(shape))
    check(q, kp, vp, k_fp, v_fp, min(41, shape[5]))


@pytest.mark.parametrize("L", [2, 33, 200])
@pytest.mark.parametrize("dtype", [HALF, BF16])
def test_masks(dtype, L):
    """Padded requests: -inf, the type's lowest value, ordinary biases, a row that sees nothing; masked keys and values that are not numbers."""
    B, t_sys = 5, 41
    q, kp, vp, k_fp, v_fp = make(B, 8, 2, L, 192, 60, dtype, seed=L)
    n = 192 + 60 + L
    mask = torch.zeros(B, n, dtype=dtype, device="cuda")
    mask[0, 10:100] = -math.inf
    mask[1, t_sys + 192:n - L] = torch.finfo(dtype).min
    mask[2] = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    mask[3] = -math.inf
    mask[4] = torch.finfo(dtype).min
    k_fp[0, :, 10:40] = math.nan                     # tokens in front of the visual span
    v_fp[0, :, 10:40] = math.inf
    for pack in (kp, vp):
        pack[1][3], pack[2][3] = math.nan, math.inf
    # the first 59 visual tokens of row 0 are masked: whole groups may hold anything
    kp[1][0, :, :, 0] = math.nan
    vp[2][0, :, :32] = -math.inf
    out, lse, w = check(q, kp, vp, k_fp, v_fp, t_sys, mask)
    assert not out[3].any() and torch.isneginf(lse[3]).all() and not w[0][3].any() and not w[1][3].any()
    check(q, kp, vp, k_fp, v_fp, t_sys, mask.view(B, 1, 1, n).float())       # another shape and type of the same numbers


@pytest.mark.parametrize("dtype", [HALF, BF16])
@pytest.mark.parametrize("shape", [(2, 8, 2, 385, 160, 70), (1, 16, 2, 200, 416, 87), (1, 32, 1, 45, 96, 33), (1, 2, 2, 1300, 0, 40), (1, 12, 2, 333, 1312, 0)], ids=str)
def test_many_row_blocks(shape, dtype):
    """Six row blocks and more: key tiles unpacked once; a live count that ends inside the first of the tiles; masks."""
    q, kp, vp, k_fp, v_fp = make(*shape, dtype, seed=sum(shape))
    check(q, kp, vp, k_fp, v_fp, min(41, shape[5]))
    t_fp = k_fp.shape[2]
    for live in (t_fp - 3, shape[3] // 2, 1):
        k_fp[:, :, live:], v_fp[:, :, live:] = math.nan, math.nan
        check(q, kp, vp, k_fp, v_fp, min(41, shape[5]), t_fp=t_fp, t_fp_dev=torch.tensor([live], dtype=torch.int32, device="cuda"), live=live)


@pytest.mark.parametrize("dtype", [HALF, BF16])
def test_masks_of_many_row_blocks(dtype):
    test_masks(dtype, 390)


@pytest.mark.parametrize("L,B", [(500, 1), (390, 2)])
def test_many_row_blocks_captured(L, B):
    test_captured_and_replayed(L, B)


@pytest.mark.parametrize("live", [70, 41, 7, 3, 0])
def test_live_count(live):
    """Tokens that are not live yet hold anything; fewer live tokens than new ones leave the first queries the visual span alone."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(2, 8, 2, 7, 96, 64, BF16, seed=live, cap=100)
    k_fp[:, :, live:] = math.nan
    v_fp[:, :, live:] = math.nan
    counter = torch.tensor([live], dtype=torch.int32, device="cuda")
    check(q, kp, vp, k_fp, v_fp, 41, t_fp=90, t_fp_dev=counter, live=live)
    if live:
        out = ops.chunk_attention(q[:, :1], None, None, k_fp, v_fp, 41, t_fp_dev=counter)
        want, _, room, _ = ref.attention64(q[:, :1], None, None, k_fp, v_fp, 41, live=live)
        assert ref.within(out, want, room)


@pytest.mark.parametrize("L", [1, 3])
@pytest.mark.parametrize("cap", [1500, 5000])
@pytest.mark.parametrize("dtype", [HALF, BF16])
def test_few_rows_of_a_long_capacity(dtype, cap, L):
    """Single tokens whose blocks merge as a cluster (1500: seven blocks a head) or by a second launch (5000): a small live count leaves most
    blocks without a key, and a row without any key has none in all of them."""
    q, kp, vp, k_fp, v_fp = make(2, 8, 2, L, 96, 700, dtype, seed=cap + L, cap=cap)
    none = torch.zeros(2, 96 + cap, dtype=dtype, device="cuda")
    none[1] = -math.inf
    for live in (cap, 700, 300, 2):
        k_fp[:, :, live:], v_fp[:, :, live:] = math.nan, math.nan
        counter = torch.tensor([live], dtype=torch.int32, device="cuda")
        for mask in (None, none):
            out, lse, w = check(q, kp, vp, k_fp, v_fp, 41, mask, t_fp=cap, t_fp_dev=counter, live=live)
        assert not out[1].any() and torch.isneginf(lse[1]).all() and not w[0][1].any()


@pytest.mark.parametrize("dtype", [HALF, BF16])
def test_offsets_and_ends_of_the_range(dtype):
    """Keys far from zero beside their spread (several times the group's range), constant groups, large and tiny ones."""
    q, kp, vp, k_fp, v_fp = make(1, 8, 2, 9, 128, 30, dtype, seed=5, offset=20.0)
    check(q, kp, vp, k_fp, v_fp, 20)
    q, kp, vp, k_fp, v_fp = make(1, 8, 2, 9, 128, 30, dtype, seed=6)
    kp[1][:, :, 5] = 0                                                    # constant groups: code 0 or not, the value is the minimum
    big = 4000.0 if dtype == HALF else 1e30
    kp[1][:, :, 6], kp[2][:, :, 6] = big, -7 * big
    q[..., 6] = (1.0 if dtype == HALF else 1.5) / big
    kp[1][:, :, 7] = torch.finfo(dtype).tiny
    check(q, kp, vp, k_fp, v_fp, 20)


def test_layouts():
    """Strided queries and caches, an unaligned one, an output of the caller's, packs that are not contiguous."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(2, 8, 2, 21, 160, 50, HALF, seed=3)
    want = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 41, return_lse=True)
    w = ops.key_weights(q, want[1], kp, k_fp, 41)

    def same(got, q=q, kp=kp, k_fp=k_fp):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        again = ops.key_weights(q, want[1], kp, k_fp, 41)
        assert torch.equal(again[0], w[0]) and torch.equal(again[1], w[1])

    q2 = q.transpose(1, 2).contiguous().transpose(1, 2)
    same(ops.chunk_attention(q2, kp, vp, k_fp, v_fp, 41, return_lse=True), q=q2)
    q3 = torch.randn(2, 21, 8, 160, device="cuda").half()[..., 8:136].copy_(q)
    same(ops.chunk_attention(q3, kp, vp, k_fp, v_fp, 41, return_lse=True), q=q3)
    q4 = torch.empty(q.numel() + 1, dtype=HALF, device="cuda")[1:].view_as(q).copy_(q).transpose(0, 0)
    same(ops.chunk_attention(q4.clone(), kp, vp, k_fp, v_fp, 41, return_lse=True))
    big = [torch.empty(2, 2, 200, 128, dtype=HALF, device="cuda") for _ in range(2)]
    for b, t in zip(big, (k_fp, v_fp)):
        b[:, :, :71] = t
    same(ops.chunk_attention(q, kp, vp, *big, 41, t_fp=71, return_lse=True))
    k5, v5 = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (k_fp, v_fp))
    same(ops.chunk_attention(q, kp, vp, k5, v5, 41, return_lse=True), k_fp=k5)
    odd = [torch.stack([t, t], -1)[..., 0] for t in kp], [torch.stack([t, t], -1)[..., 0] for t in vp]
    same(ops.chunk_attention(q, *odd, k_fp, v_fp, 41, return_lse=True), kp=odd[0])
    o = torch.full((2, 21, 16, 128), 7.0, dtype=HALF, device="cuda")
    got = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 41, out=o[:, :, 4:12], return_lse=True)
    assert got[0].data_ptr() == o[:, :, 4:12].data_ptr()
    same(got)
    assert (o[:, :, :4] == 7).all() and (o[:, :, 12:] == 7).all()


def test_weights_add_up():
    """In place, into room for more keys than there are, and twice the same numbers."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(2, 8, 2, 40, 96, 50, BF16, seed=8)
    _, lse = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 41, return_lse=True)
    one = ops.key_weights(q, lse, kp, k_fp, 41)
    assert abs(float(one[0].sum() + one[1].sum()) / (2 * 8 * 40) - 1) < 1e-4        # the probabilities of a row sum to one
    base = (torch.rand(2, 2, 96, device="cuda"), torch.rand(2, 2, 120, device="cuda"))
    acc = tuple(t.clone() for t in base)
    got = ops.key_weights(q, lse, kp, k_fp, 41, weights=acc, out=acc)
    assert got[0].data_ptr() == acc[0].data_ptr()
    assert torch.equal(acc[0], base[0] + one[0]) and torch.equal(acc[1][..., :90], base[1][..., :90] + one[1])
    assert torch.equal(acc[1][..., 90:], base[1][..., 90:])
    fresh = ops.key_weights(q, lse, kp, k_fp, 41, weights=base)
    assert torch.equal(fresh[0], acc[0]) and torch.equal(fresh[1], acc[1])


def test_agrees_with_the_decode_step():
    """One token on the same cache: the framework's single-token step without calibration (which rounds where the reference does)."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(4, 32, 8, 1, 1312, 77, HALF, seed=9)
    a = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 41)
    b = ops.decode_attention(q.transpose(1, 2), kp, vp, k_fp, v_fp, 41, 4, calibrate=False)
    err = (a.double() - b.transpose(1, 2).double()).norm() / b.double().norm()
    assert err < 1e-2


@pytest.mark.parametrize("L,B", [(1, 2), (9, 1), (40, 2), (300, 1)])
def test_captured_and_replayed(L, B):
    """Both calls in a CUDA graph whose inputs and live count change between replays, beside eager calls on another stream."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(B, 8, 2, L, 160, 100, BF16, seed=L, cap=500)
    counter = torch.tensor([100 + L], dtype=torch.int32, device="cuda")
    acc = (torch.zeros(B, 2, 160, device="cuda"), torch.zeros(B, 2, 500, device="cuda"))

    def both():
        out, lse = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 41, t_fp_dev=counter, return_lse=True)
        ops.key_weights(q, lse, kp, k_fp, 41, weights=acc, out=acc, t_fp_dev=counter)
        return out, lse
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = both()
    for step, live in enumerate((100 + L, 300, 450)):
        counter.fill_(live)
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)))
        for t in acc:
            t.zero_()
        graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            again = both()
            again_acc = [t.clone() for t in acc]
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
        assert all(torch.equal(2 * t, u) for t, u in zip(ops.key_weights(q, lse, kp, k_fp, 41, t_fp_dev=counter), again_acc))
        want, want_l, room, room_l = ref.attention64(q, kp, vp, k_fp, v_fp, 41, live=min(live, 500))      # a count above the capacity is the capacity
        assert ref.within(out, want, room) and ref.within(lse, want_l, room_l)


def test_two_streams_at_once():
    """Calls that overlap on two streams have workspaces of their own; results do not depend on when they run."""
    from calibquant_b200 import ops
    cases = [make(4, 8, 2, L, 1312, 100, HALF, seed=L) for L in (1, 60, 700)]
    want = [ops.chunk_attention(q, kp, vp, k, v, 41, return_lse=True) for q, kp, vp, k, v in cases]
    want_w = [ops.key_weights(c[0], w[1], c[1], c[3], 41) for c, w in zip(cases, want)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for rep in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                for (q, kp, vp, k, v), w in zip(cases, want):
                    got.append((ops.chunk_attention(q, kp, vp, k, v, 41, return_lse=True), ops.key_weights(q, w[1], kp, k, 41)))
    torch.cuda.synchronize()
    for i, (o, w) in enumerate(got):
        assert torch.equal(o[0], want[i % 3][0]) and torch.equal(o[1], want[i % 3][1])
        assert all(torch.equal(a, b) for a, b in zip(w, want_w[i % 3]))


@pytest.mark.parametrize("L", [2, 70, 260])
def test_offsets_past_32_bits(L):
    """The second request's full-precision tokens lie more than 2^31 elements behind the first one's."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(2, 4, 1, L, 64, 40, BF16, seed=L)
    n, far = k_fp.shape[2], 2 ** 31 + 2 ** 20
    views = []
    for t in (k_fp, v_fp):
        big = torch.empty(far + n * 128, dtype=BF16, device="cuda").as_strided((2, 1, n, 128), (far, n * 128, 128, 1))
        views.append(big.copy_(t))
    a, la = ops.chunk_attention(q, kp, vp, *views, 41, return_lse=True)
    b, lb = ops.chunk_attention(q, kp, vp, k_fp, v_fp, 41, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    assert all(torch.equal(x, y) for x, y in zip(ops.key_weights(q, la, kp, views[0], 41), ops.key_weights(q, lb, kp, k_fp, 41)))


def test_many_small_requests():
    """More (request, head) pairs than a launch has SMs, one key each."""
    q, kp, vp, k_fp, v_fp = make(70, 8, 8, 1, 0, 0, HALF, seed=4)
    check(q, kp, vp, k_fp, v_fp, 0)
    q, kp, vp, k_fp, v_fp = make(40, 16, 4, 2, 32, 1, BF16, seed=4)
    check(q, kp, vp, k_fp, v_fp, 1)


def test_empty_batch():
    from calibquant_b200 import ops
    q, k = torch.empty(0, 3, 8, 128, dtype=HALF, device="cuda"), torch.empty(0, 2, 9, 128, dtype=HALF, device="cuda")
    out, lse = ops.chunk_attention(q, None, None, k, k, 4, return_lse=True)
    assert out.shape == q.shape and lse.shape == (0, 8, 3)
    assert [t.shape for t in ops.key_weights(q, lse, None, k, 4)] == [(0, 2, 0), (0, 2, 9)]


def test_no_queries():
    """Nothing to attend: an empty result, weights as they were."""
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(2, 8, 2, 1, 64, 20, HALF)
    out, lse = ops.chunk_attention(q[:, :0], kp, vp, k_fp, v_fp, 4, return_lse=True)
    assert out.shape == (2, 0, 8, 128) and lse.shape == (2, 8, 0)
    fresh = ops.key_weights(q[:, :0], lse, kp, k_fp, 4)
    assert not fresh[0].any() and not fresh[1].any() and fresh[1].shape == (2, 2, 21)
    w = (torch.rand(2, 2, 64, device="cuda"), torch.rand(2, 2, 30, device="cuda"))
    for got in (ops.key_weights(q[:, :0], lse, kp, k_fp, 4, weights=w), ops.key_weights(q[:, :0], lse, kp, k_fp, 4, weights=w, out=w)):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_refusals():
    from calibquant_b200 import ops
    q, kp, vp, k_fp, v_fp = make(1, 8, 2, 3, 64, 20, HALF)
    lse = torch.zeros(1, 8, 3, device="cuda")
    f = lambda **k: ops.chunk_attention(**{**dict(q=q, k_pack=kp, v_pack=vp, k_fp=k_fp, v_fp=v_fp, t_sys=4), **k})
    w = lambda **k: ops.key_weights(**{**dict(q=q, lse=lse, k_pack=kp, k_fp=k_fp, t_sys=4), **k})
    both = [dict(q=q.float()), dict(q=q.bfloat16()), dict(q=q[0]), dict(k_fp=k_fp[0]), dict(k_fp=k_fp[..., :64]), dict(bits=2), dict(group_size=64),
            dict(t_fp=2), dict(t_fp=24), dict(t_sys=-1), dict(mask=torch.zeros(1, 86, device="cuda")), dict(k_pack=kp[:2]),
            dict(k_pack=(kp[0], kp[1], kp[2][..., :1])), dict(k_pack=(kp[0].long(), kp[1], kp[2])), dict(q=q[:, :, :7]),
            dict(t_fp_dev=torch.tensor([5], device="cuda"))]
    for kw in both:
        for call in (f, w):
            with pytest.raises((ValueError, TypeError, RuntimeError, AssertionError)):
                call(**kw)
    for kw in (dict(v_pack=None), dict(v_pack=kp), dict(v_fp=v_fp[:, :, :9]), dict(out=torch.empty(1, 3, 8, 128, device="cuda")), dict(v_fp=v_fp.cpu()),
               dict(out=torch.empty(1, 3, 8, 130, dtype=HALF, device="cuda")[..., :128])):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            f(**kw)
    z = lambda *s: torch.zeros(*s, device="cuda")
    for kw in (dict(lse=lse.half()), dict(lse=lse[..., :2]), dict(weights=(z(1, 2, 64), z(1, 2, 22))), dict(weights=(z(1, 2, 32), z(1, 2, 23))),
               dict(weights=(z(1, 2, 64), z(1, 2, 30)), out=(z(1, 2, 64), z(1, 2, 31))), dict(weights=z(1, 2, 64)),
               dict(out=(z(1, 2, 64), z(1, 2, 30).double()))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            w(**kw)
    with pytest.raises(RuntimeError):
        ops.chunk_attention(q.cpu(), kp, vp, k_fp, v_fp, 4)
