"""The C entry points of the chunk attention, the key weights and the evictions refuse bad arguments on the host, before any CUDA call."""

import ctypes

import pytest

from calibquant_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.lib()


@pytest.fixture(scope="module")
def p16():
    buf = ctypes.create_string_buffer(4096)
    p16.keep = buf
    return (ctypes.addressof(buf) + 15) // 16 * 16


def chunk_args(p, **changes):
    a = _lib.ChunkArgs()
    a.batch, a.n_q_heads, a.n_kv_heads, a.head_dim, a.q_len, a.t_vis, a.t_fp, a.t_sys = 1, 8, 2, 128, 3, 64, 10, 4
    a.bits, a.group_size, a.dtype = 4, 32, _lib.CQ_DTYPE_BF16
    for name in ("q", "k_code", "k_scale", "k_mn", "v_code", "v_scale", "v_mn", "k_fp", "v_fp", "out", "lse"):
        setattr(a, name, p)
    a.q_strides = a.out_strides = (ctypes.c_int64 * 3)(4096, 1024, 128)
    a.fp_stride_b, a.fp_stride_h = 2 * 1280, 1280
    for name, value in changes.items():
        setattr(a, name, (ctypes.c_int64 * 3)(*value) if name.endswith("strides") else value)
    return a


BAD = [dict(batch=-1), dict(n_q_heads=7), dict(n_kv_heads=0), dict(q_len=0), dict(q_len=11), dict(t_vis=-32), dict(t_sys=11), dict(reserved=1), dict(dtype=2),
       dict(q=None), dict(k_fp=None), dict(k_scale=None), dict(fp_stride_h=1284), dict(q_strides=(4096, 1024, 127)), dict(q_strides=(4096, 0, 128)),
       dict(q_strides=(4096, -1024, 128)), dict(q_strides=(4096, 1024, 0))]
UNSUPPORTED = [dict(head_dim=64), dict(group_size=64), dict(bits=2), dict(bits=8), dict(t_vis=65), dict(n_q_heads=258, n_kv_heads=2)]


@pytest.mark.parametrize("changes", BAD, ids=str)
def test_bad_arguments(lib, p16, changes):
    a = chunk_args(p16, **changes)
    assert lib.cq_chunk_attn_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.cq_chunk_attn(ctypes.byref(a), p16, 1 << 30, None) == _lib.CQ_ERR_BAD_ARG
    assert lib.cq_key_weights_workspace_bytes(ctypes.byref(a), 16) == 0
    assert lib.cq_key_weights(ctypes.byref(a), None, None, p16, p16, 16, p16, 1 << 30, None) == _lib.CQ_ERR_BAD_ARG


@pytest.mark.parametrize("changes", UNSUPPORTED, ids=str)
def test_unsupported(lib, p16, changes):
    a = chunk_args(p16, **changes)
    assert lib.cq_chunk_attn_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.cq_chunk_attn(ctypes.byref(a), p16, 1 << 30, None) == _lib.CQ_ERR_UNSUPPORTED
    assert lib.cq_key_weights(ctypes.byref(a), None, None, p16, p16, 16, p16, 1 << 30, None) == _lib.CQ_ERR_UNSUPPORTED


def test_each_call_on_its_own(lib, p16):
    ref = lambda **c: ctypes.byref(chunk_args(p16, **c))
    for c in (dict(out=None), dict(v_fp=None), dict(v_code=None), dict(out=p16 + 2), dict(out_strides=(4096, 1024, 4))):
        assert lib.cq_chunk_attn(ref(**c), p16, 1 << 30, None) == _lib.CQ_ERR_BAD_ARG
    assert lib.cq_chunk_attn(None, p16, 1 << 30, None) == _lib.CQ_ERR_BAD_ARG
    need = lib.cq_chunk_attn_workspace_bytes(ref())
    assert need >= 256
    assert lib.cq_chunk_attn(ref(), p16, need - 1, None) == _lib.CQ_ERR_WORKSPACE
    assert lib.cq_chunk_attn(ref(), None, need, None) == _lib.CQ_ERR_WORKSPACE
    assert lib.cq_chunk_attn(ref(batch=0), p16, 1 << 30, None) == _lib.CQ_OK
    w = lambda a, vis=p16, fp=p16, cap=16, ws=p16, n=1 << 30: lib.cq_key_weights(a, None, None, vis, fp, cap, ws, n, None)
    assert w(ref(lse=None)) == w(ref(), vis=None) == w(ref(), fp=None) == w(ref(), cap=9) == _lib.CQ_ERR_BAD_ARG
    assert w(ref(), ws=None) == w(ref(), n=8) == _lib.CQ_ERR_WORKSPACE
    assert w(ref(), cap=1 << 31) == _lib.CQ_ERR_UNSUPPORTED
    assert w(ref(batch=0)) == _lib.CQ_OK


def test_evictions(lib, p16):
    def groups(t_vis=64, keep=1, bits=4, group=32, dim=128, batch=1, heads=1, p=p16, w=p16):
        return lib.cq_evict_groups(p, p16, p16, p16, p16, p16, w, batch, heads, dim, t_vis, keep, bits, group, p16, p16, p16, p16, p16, p16, p16, p16, None)
    assert groups(batch=0) == _lib.CQ_OK
    for kw in (dict(t_vis=0), dict(t_vis=65), dict(keep=0), dict(keep=3), dict(batch=-1), dict(heads=0), dict(p=None), dict(w=p16 + 4)):
        assert groups(**kw) == _lib.CQ_ERR_BAD_ARG
    for kw in (dict(bits=3), dict(bits=8), dict(group=64), dict(dim=64), dict(t_vis=32 * 16385), dict(batch=256, heads=256)):
        assert groups(**kw) == _lib.CQ_ERR_UNSUPPORTED

    def tokens(t=50, keep=20, sys=5, recent=5, sb=6400, sh=6400, ws=50, batch=1, dim=128, k=p16, w=p16):
        return lib.cq_evict_tokens(k, p16, sb, sh, w, ws, batch, 1, dim, t, keep, sys, recent, p16, p16, p16, p16, None)
    assert tokens(batch=0) == _lib.CQ_OK
    for kw in (dict(t=0), dict(keep=0), dict(keep=51), dict(sys=16), dict(sys=-1), dict(recent=-1), dict(recent=2 ** 31 - 1), dict(sb=6404), dict(sh=2), dict(ws=49),
               dict(k=None), dict(k=p16 + 8), dict(w=None), dict(batch=-1)):
        assert tokens(**kw) == _lib.CQ_ERR_BAD_ARG
    for kw in (dict(dim=64), dict(t=24577, ws=24577)):
        assert tokens(**kw) == _lib.CQ_ERR_UNSUPPORTED


def test_what_is_narrower_than_16_bytes(lib, p16):
    """Pointers to 4- and 8-byte numbers may start anywhere that their type may."""
    w = lambda a, vis_in=None, fp_in=None, vis=p16, fp=p16: lib.cq_key_weights(a, vis_in, fp_in, vis, fp, 16, p16, 1 << 30, None)
    for c in (dict(lse=p16 + 2), dict(t_fp_dev=p16 + 1)):
        assert lib.cq_chunk_attn(ctypes.byref(chunk_args(p16, **c)), p16, 1 << 30, None) == _lib.CQ_ERR_BAD_ARG
        assert w(ctypes.byref(chunk_args(p16, **c))) == _lib.CQ_ERR_BAD_ARG
    for kw in (dict(vis_in=p16 + 2), dict(fp_in=p16 + 1), dict(vis=p16 + 2), dict(fp=p16 + 3)):
        assert w(ctypes.byref(chunk_args(p16, batch=0)), **kw) == _lib.CQ_ERR_BAD_ARG
    assert w(ctypes.byref(chunk_args(p16, batch=0, lse=p16 + 4, t_fp_dev=p16 + 4)), vis=p16 + 4) == _lib.CQ_OK

    def tokens(w=p16, w_out=p16, kept=p16):
        return lib.cq_evict_tokens(p16, p16, 6400, 6400, w, 50, 0, 1, 128, 50, 20, 5, 5, p16, p16, w_out, kept, None)
    assert tokens(w=p16 + 4, w_out=p16 + 4, kept=p16 + 8) == _lib.CQ_OK
    for kw in (dict(w=p16 + 2), dict(w_out=p16 + 2), dict(kept=p16 + 4)):
        assert tokens(**kw) == _lib.CQ_ERR_BAD_ARG
