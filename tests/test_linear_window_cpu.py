"""What linear attention and window attention refuse, before anything is launched."""

import ctypes

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import (_abi, linear_attention, linear_attention_step, window_attention, window_attention_step,
                                        window_cache_write)

D, P, MIS = 128, 0x10000, 0x10002
BF16 = torch.bfloat16


def Z(*shape, **kw):
    return torch.zeros(*shape, **kw)


# ---------------------------------------------------------------------------
# Linear attention
# ---------------------------------------------------------------------------

def _linear(**kw):
    return {**dict(q=Z(1, 4, 1, D), k=Z(1, 4, 1, D), v=Z(1, 4, 2, D), g=Z(2)), **kw}


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(k=Z(1, 4, 2, D))), (ValueError, dict(v=Z(1, 5, 2, D))), (ValueError, dict(q=Z(4, 1, D))),
    (ValueError, dict(q=Z(1, 4, 1, 64), k=Z(1, 4, 1, 64))), (ValueError, dict(v=Z(1, 4, 2, 64))),
    (ValueError, dict(q=Z(1, 4, 3, D), k=Z(1, 4, 3, D))), (ValueError, dict(q=Z(1, 4, 0, D), k=Z(1, 4, 0, D))),
    (ValueError, dict(g=Z(1))), (ValueError, dict(g=Z(1, 4, 2))), (ValueError, dict(v=Z(1, 4, 2, D, dtype=BF16))),
    (TypeError, dict(g=Z(2, dtype=BF16))), (TypeError, dict(g=Z(2, dtype=torch.float64))),
    (TypeError, {n: Z(1, 4, 2, D).half() for n in "qkv"}),
    (ValueError, dict(cu_seqlens=torch.tensor([0]))), (ValueError, dict(cu_seqlens=torch.tensor([0., 4.]))),
    (ValueError, dict(cu_seqlens=torch.tensor([[0, 4]]))), (ValueError, dict(initial_state=Z(2, 2, D, D))),
    (ValueError, dict(initial_state=Z(1, 2, D, D, dtype=BF16))),
    (ValueError, dict(cu_seqlens=torch.tensor([0, 2, 4]), initial_state=Z(1, 2, D, D))),
    (ValueError, dict(q=Z(2, 4, 1, D), k=Z(2, 4, 1, D), v=Z(2, 4, 2, D), cu_seqlens=torch.tensor([0, 4]))),
    (RuntimeError, {})])                         # right, but on the CPU
def test_linear_refuses(error, kw):
    with pytest.raises(error):
        linear_attention(**_linear(**kw))


def _linear_step(N=3, slots=4, **kw):
    return {**dict(q=Z(N, 1, D), k=Z(N, 1, D), v=Z(N, 2, D), g=Z(2), state=Z(slots, 2, D, D)), **kw}


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(q=Z(3, D))), (ValueError, dict(g=Z(3, 2))), (TypeError, dict(g=Z(2).half())), (ValueError, dict(state=Z(2, 2, D, D))),
    (ValueError, dict(state=Z(4, 1, D, D))), (ValueError, dict(state=Z(4, 2, D, D, dtype=BF16))),
    (ValueError, dict(state=Z(4, 2, D, D).transpose(2, 3))), (ValueError, dict(state=Z(1, 2, D, D).expand(4, 2, D, D))),
    (ValueError, dict(state=Z(4 * 2 * D * D + 1)[1:].view(4, 2, D, D))),
    (ValueError, dict(state=Z(5 * D * D).as_strided((4, 2, D, D), (D * D, D * D, D, 1)))),
    (ValueError, dict(state_indices=Z(2, dtype=torch.int32))), (ValueError, dict(state_indices=Z(3))),
    (RuntimeError, dict(v=Z(3, 2, D, requires_grad=True))), (RuntimeError, dict(g=Z(2, requires_grad=True))), (RuntimeError, {})])
def test_linear_step_refuses(error, kw):
    with pytest.raises(error):
        linear_attention_step(**_linear_step(**kw))


# ---------------------------------------------------------------------------
# Window attention
# ---------------------------------------------------------------------------

def _window(**kw):
    return {**dict(q=Z(1, 4, 2, D), k=Z(1, 4, 1, D), v=Z(1, 4, 1, D), window=3, sinks=1), **kw}


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(v=Z(1, 4, 2, D))), (ValueError, dict(q=Z(1, 5, 2, D))), (ValueError, dict(q=Z(4, 2, D))),
    (ValueError, dict(q=Z(1, 4, 2, 64))), (ValueError, dict(k=Z(1, 4, 1, 64), v=Z(1, 4, 1, 64))),
    (ValueError, dict(k=Z(1, 4, 3, D), v=Z(1, 4, 3, D))), (ValueError, dict(k=Z(1, 4, 0, D), v=Z(1, 4, 0, D))),
    (ValueError, dict(q=Z(1, 4, 0, D))), (ValueError, dict(q=Z(1, 4, 2, D, dtype=BF16))),
    (TypeError, {n: Z(1, 4, 2, D).half() for n in "qkv"}),
    (ValueError, dict(window=0)), (ValueError, dict(window=-5)), (ValueError, dict(window=2.0)), (ValueError, dict(window=True)),
    (ValueError, dict(window=1 << 30)), (ValueError, dict(sinks=-1)), (ValueError, dict(sinks=1.5)), (ValueError, dict(sinks=False)),
    (ValueError, dict(window=1 << 29, sinks=1 << 29)),
    (ValueError, dict(cu_seqlens=torch.tensor([0]))), (ValueError, dict(cu_seqlens=torch.tensor([0., 4.]))),
    (ValueError, dict(cu_seqlens=torch.tensor([[0, 4]]))),
    (ValueError, dict(q=Z(2, 4, 2, D), k=Z(2, 4, 1, D), v=Z(2, 4, 1, D), cu_seqlens=torch.tensor([0, 4]))),
    (RuntimeError, {})])
def test_window_refuses(error, kw):
    with pytest.raises(error):
        window_attention(**_window(**kw))


_CACHE = [
    (ValueError, dict(k_cache=Z(4, 8, 2, D))), (ValueError, dict(v_cache=Z(4, 8, D))), (ValueError, dict(k_cache=Z(4, 8, 1, D, dtype=BF16))),
    (ValueError, dict(v_cache=Z(5, 8, 1, D))), (ValueError, dict(k_cache=Z(4, 8, 1, 2 * D)[..., ::2])),
    (ValueError, dict(k_cache=Z(1, 8, 1, D).expand(4, 8, 1, D))), (ValueError, dict(v_cache=Z(4 * 8 * D + 1)[1:].view(4, 8, 1, D))),
    (ValueError, dict(k_cache=Z(12 * D).as_strided((4, 8, 1, D), (D, D, D, 1)))),
    (RuntimeError, dict(k_cache=Z(4, 8, 1, D, requires_grad=True)))]


def _write(**kw):
    return {**dict(k=Z(3, 5, 1, D), v=Z(3, 5, 1, D), k_cache=Z(4, 8, 1, D), v_cache=Z(4, 8, 1, D), sinks=2), **kw}


@pytest.mark.parametrize("error,kw", _CACHE + [
    (ValueError, dict(k=Z(3, 5, D))), (ValueError, dict(v=Z(3, 4, 1, D))), (ValueError, dict(v=Z(3, 5, 1, D, dtype=BF16))),
    (ValueError, dict(sinks=8)), (ValueError, dict(sinks=-1)), (ValueError, dict(positions=Z(2, dtype=torch.int64))),
    (ValueError, dict(positions=Z(3))), (ValueError, dict(cache_indices=Z(3, 1, dtype=torch.int32))),
    (ValueError, dict(k=Z(5, 1, 1, D), v=Z(5, 1, 1, D))), (ValueError, dict(cu_seqlens=torch.tensor([0, 5]))),
    (ValueError, dict(k=Z(1, 5, 1, D), v=Z(1, 5, 1, D), cu_seqlens=torch.tensor([0, 2, 5]), positions=Z(1, dtype=torch.int64))),
    (RuntimeError, dict(k=Z(3, 5, 1, D, requires_grad=True))), (RuntimeError, {})])
def test_cache_write_refuses(error, kw):
    with pytest.raises(error):
        window_cache_write(**_write(**kw))


def _step(**kw):
    return {**dict(q=Z(3, 2, D), k=Z(3, 1, D), v=Z(3, 1, D), k_cache=Z(4, 8, 1, D), v_cache=Z(4, 8, 1, D),
                   positions=Z(3, dtype=torch.int64), window=6, sinks=2), **kw}


@pytest.mark.parametrize("error,kw", _CACHE + [
    (ValueError, dict(q=Z(3, D))), (ValueError, dict(k=None)), (ValueError, dict(v=None)), (ValueError, dict(q=Z(2, 2, D))),
    (ValueError, dict(k=None, v=None, q=Z(3, D))), (ValueError, dict(k=None, v=None, q=Z(3, 2, 64))), (ValueError, dict(k=Z(3, 1, D, dtype=BF16))),
    (ValueError, dict(window=7)), (ValueError, dict(sinks=3)), (ValueError, dict(window=0)), (ValueError, dict(positions=Z(2, dtype=torch.int64))),
    (ValueError, dict(positions=Z(3))), (ValueError, dict(cache_indices=Z(2, dtype=torch.int32))),
    (ValueError, dict(q=Z(5, 2, D), k=Z(5, 1, D), v=Z(5, 1, D), positions=Z(5, dtype=torch.int32))),
    (RuntimeError, dict(q=Z(3, 2, D, requires_grad=True))), (RuntimeError, {}), (RuntimeError, dict(k=None, v=None))])
def test_window_step_refuses(error, kw):
    with pytest.raises(error):
        window_attention_step(**_step(**kw))


def test_caches_that_are_one_refused():
    c = Z(4, 8, 1, D)
    with pytest.raises(ValueError, match="same memory"):
        window_cache_write(**_write(k_cache=c, v_cache=c))
    with pytest.raises(ValueError, match="same memory"):
        window_attention_step(**_step(k_cache=c, v_cache=c))


def test_caches_side_by_side_and_by_head():
    """Keys and values in one allocation, and caches laid out by head, pass the checks (and end at the one for a GPU)."""
    both = Z(4, 8, 2, 1, D)
    heads = [Z(4, 1, 8, D).transpose(1, 2) for _ in range(2)]
    for kc, vc in ((both[:, :, 0], both[:, :, 1]), heads):
        with pytest.raises(RuntimeError, match="GPU|cuda|CUDA|device"):
            window_attention_step(**_step(k_cache=kc, v_cache=vc))


def test_caches_of_too_many_rows():
    big = [torch.empty(1, 1 << 30, 1, D, device="meta", dtype=BF16) for _ in range(2)]
    with pytest.raises(ValueError, match="rows"):
        window_cache_write(Z(1, 1, 1, D, dtype=BF16), Z(1, 1, 1, D, dtype=BF16), *big)


# ---------------------------------------------------------------------------
# The C entries: a status, nothing enqueued (the addresses are never dereferenced)
# ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    return _abi.load()


def _linear_c(lib, backward=False, **kw):
    a = _abi.LinearArgs(B=2, T=1000, N=2, Hk=1, Hv=2, d=128, dtype=1, scale=0.1, g_sh=1)
    for n in ("q", "k", "v", "g", "o", "ws", "saved", "dout", "dq", "dk", "dv", "dg"):
        setattr(a, n, P)
    for n in ("q", "k", "v", "do"):
        setattr(a, n + "_sb", 256000), setattr(a, n + "_st", 256), setattr(a, n + "_sh", 128)
    a.ws_bytes = lib.gsa_linear_attn_workspace_bytes(2, 1000, 2, 0, 1, 2, 1, int(backward))
    a.saved_bytes = lib.gsa_linear_attn_saved_bytes(2, 1000, 2, 0, 1, 2, 1)
    assert a.saved_bytes > 0 and a.ws_bytes >= 2 * a.saved_bytes          # in segments
    for n, x in kw.items():
        setattr(a, n, x)
    return (lib.gsa_linear_attn_backward if backward else lib.gsa_linear_attn)(ctypes.byref(a), None)


def test_c_linear_refusals(lib):
    assert lib.gsa_linear_attn(None, None) == lib.gsa_linear_attn_backward(None, None) == 1
    for back in (False, True):
        for n in ("q", "k", "v", "g", "ws") + (("saved", "dout", "dq", "dk", "dv") if back else ("o",)):
            assert _linear_c(lib, back, **{n: None}) == 1, n
        assert _linear_c(lib, back, dtype=2) == 3
        for kw in (dict(B=0), dict(T=0), dict(N=3), dict(Hk=0), dict(Hk=3), dict(Hv=1 << 24), dict(d=64), dict(ws_bytes=1024),
                   dict(saved_bytes=1024), dict(cu_seqlens=P, cu_bytes=4), dict(cu_seqlens=P, cu_bytes=2, B=1), dict(q_st=-256),
                   dict(k_st=1 << 24)):
            assert _linear_c(lib, back, **kw) == 2, kw
        for kw in (dict(q=P + 8), dict(k_st=257), dict(v_sb=4), dict(k_sh=132), dict(g=MIS), dict(ws=P + 8), dict(state_in=P + 4),
                   dict(state_out=P + 4), dict(cu_seqlens=P + 2, cu_bytes=4, B=1, N=2)):
            assert _linear_c(lib, back, **kw) == 4, kw
    assert _linear_c(lib, True, do_st=4) == _linear_c(lib, True, dg=MIS) == _linear_c(lib, True, dstate_in=P + 8) == 4


def test_c_linear_sizes(lib):
    refused, last = ctypes.c_size_t(-1).value, 2 ** 31 - 1
    for back in (0, 1):
        def f(*a):
            return lib.gsa_linear_attn_workspace_bytes(*a, back)
        for bad in ((0, 5, 1, 0, 1, 1, 1), (1, 0, 1, 0, 1, 1, 1), (1, 5, 0, 1, 1, 1, 1), (1, 5, 1, 0, 0, 0, 1), (1, 5, 1, 0, 1, 1, 7),
                    (1, 5, 1, 0, 2, 3, 1), (1, last, 1, 0, 1, 1, 1), (last, last, last, 0, last, last, 1), (2 ** 29, 64, 2 ** 29, 0, 32, 32, 1)):
            assert f(*bad) == refused, bad
        for N in (2 ** 19 - 1, 2 ** 19):         # of 16 heads and one token each
            assert (f(N, 1, N, 0, 16, 16, 1) != refused) == (f(1, 1, N, 1, 16, 16, 1) != refused) == (N < 2 ** 19)
    saved = lib.gsa_linear_attn_saved_bytes
    assert lib.gsa_linear_attn_workspace_bytes(1, 64, 1, 0, 2, 2, 1, 0) == saved(1, 64, 1, 0, 2, 2, 1) == 0     # one chunk
    # a state of 64 KiB for each segment and v head: of 16 chunks of 64 where 16 heads have 16384 tokens (packed: of 8, and one
    # more begun; fp32: of 16 of 32); none for many heads
    assert saved(1, 16384, 1, 0, 16, 16, 1) == 16 * 16 * 65536
    assert saved(1, 16384, 1, 1, 16, 16, 1) == 33 * 16 * 65536 and saved(1, 16384, 1, 0, 16, 16, 0) == 32 * 16 * 65536
    assert saved(11, 16384, 11, 0, 16, 16, 1) == 0


def _linear_step_c(lib, **kw):
    a = dict(q=P, qn=128, qh=128, k=P, kn=128, kh=128, v=P, vn=256, vh=128, g=P, gh=1, idx=P, ib=4, S=P, sn=2 * D * D, sh=D * D, N=3,
             slots=4, Hk=1, Hv=2, d=128, scale=0.1, dtype=1, o=P)
    return lib.gsa_linear_step(*{**a, **kw}.values(), None)


def test_c_linear_step_refusals(lib):
    for n in ("q", "k", "v", "g", "S", "o"):
        assert _linear_step_c(lib, **{n: None}) == 1
    assert _linear_step_c(lib, dtype=5) == 3
    for kw in (dict(N=0), dict(N=65536), dict(slots=0), dict(Hk=0), dict(Hk=3), dict(Hv=65536), dict(d=64), dict(ib=2), dict(idx=None, N=5)):
        assert _linear_step_c(lib, **kw) == 2
    for kw in (dict(S=P + 4), dict(sn=2 * D * D + 1), dict(sh=D * D + 2), dict(idx=MIS), dict(g=MIS), dict(q=P + 1), dict(o=P + 1)):
        assert _linear_step_c(lib, **kw) == 4


def _window_c(lib, backward=False, **kw):
    a = _abi.WindowArgs(B=2, T=1000, N=2, H=2, Hkv=1, d=128, dtype=1, window=300, sinks=4, scale=0.1)
    for n in ("q", "k", "v", "o", "lse", "o_low", "ws", "dout", "dq", "dk", "dv"):
        setattr(a, n, P)
    for n in ("q", "k", "v", "do"):
        setattr(a, n + "_sb", 256000), setattr(a, n + "_st", 256), setattr(a, n + "_sh", 128)
    a.ws_bytes = lib.gsa_window_attn_workspace_bytes(2, 1000, 2, 0, 2, 1, 300, 4, 1)
    for n, x in kw.items():
        setattr(a, n, x)
    return (lib.gsa_window_attn_backward if backward else lib.gsa_window_attn)(ctypes.byref(a), None)


def test_c_window_refusals(lib):
    assert lib.gsa_window_attn(None, None) == lib.gsa_window_attn_backward(None, None) == 1
    for back in (False, True):
        for n in ("q", "k", "v", "o") + (("lse", "ws", "dout", "dq", "dk", "dv") if back else ()):
            assert _window_c(lib, back, **{n: None}) == 1, n
        assert _window_c(lib, back, dtype=2) == 3
        for kw in (dict(B=0), dict(T=0), dict(N=3), dict(Hkv=0), dict(Hkv=3), dict(H=65536), dict(d=64), dict(window=0), dict(sinks=-1),
                   dict(T=2 ** 31 - 1), dict(cu_seqlens=P, cu_bytes=4), dict(cu_seqlens=P, cu_bytes=2, B=1), dict(q_st=-256),
                   dict(k_st=1 << 24)):
            assert _window_c(lib, back, **kw) == 2, kw
        for kw in (dict(q=P + 8), dict(k_st=257), dict(v_sb=4), dict(k_sh=132), dict(lse=MIS), dict(o=P + 8), dict(o_low=P + 8),
                   dict(cu_seqlens=P + 2, cu_bytes=4, B=1, N=2)):
            assert _window_c(lib, back, **kw) == 4, kw
    assert _window_c(lib, True, ws_bytes=1024) == 2
    assert _window_c(lib, True, do_st=4) == _window_c(lib, True, dv=P + 8) == _window_c(lib, True, ws=P + 8) == 4


def test_c_window_sizes(lib):
    f, last = lib.gsa_window_attn_workspace_bytes, 2 ** 31 - 1
    for bad in ((0, 5, 1, 0, 1, 1, 1, 0, 1), (1, 0, 1, 0, 1, 1, 1, 0, 1), (1, 5, 1, 0, 3, 2, 1, 0, 1), (1, 5, 1, 0, 1, 1, 0, 0, 1),
                (1, 5, 1, 0, 1, 1, 1, -1, 1), (1, 5, 1, 0, 1, 1, 1, 0, 7), (1, last, 1, 0, 1, 1, 1, 0, 1),
                (last, last, last, 0, 1, 1, 1, 0, 1), (1, 2 ** 26, 1, 0, 8, 8, last, last, 1)):
        assert f(*bad) == 0, bad
    # D alone where there are no far queries: a window of everything, first tokens that are all of it, none
    assert f(1, 320, 1, 0, 2, 2, last, last, 1) == f(1, 320, 1, 0, 2, 2, 280, 40, 1) == f(1, 320, 1, 0, 2, 2, 9, 0, 1) == 320 * 2 * 4
    # near sums of 64 keys (dk and dv, fp32) and far sums of 32 keys for 3 parts of 128 queries and each head
    assert f(1, 320, 1, 0, 2, 2, 9, 4, 1) == 320 * 2 * 4 + 2 * 2 * 64 * 512 + 3 * 2 * 2 * 32 * 512
    # few blocks of keys (5 and one key head) for many tiles of queries (8 heads, 6 tiles): 12 parts for each block
    assert f(1, 320, 1, 0, 8, 1, last, 0, 1) == 320 * 8 * 4 + 5 * 12 * 2 * 64 * 512
    # many first tokens: the parts hold more queries, not the workspace more parts
    assert f(1, 65536, 1, 0, 16, 4, 100, 30000, 1) < 2 << 30


def _write_c(lib, **kw):
    a = dict(k=P, kb=1280, kt=256, kh=128, v=P, vb=1280, vt=256, vh=128, cu=None, cb=0, B=3, T=5, N=3, Hkv=2, d=128, dtype=1, pos=P, pb=8,
             idx=P, ib=4, kc=P, kcn=2048, kct=256, kch=128, vc=P, vcn=2048, vct=256, vch=128, slots=4, rows=8, sinks=2)
    return lib.gsa_window_cache_write(*{**a, **kw}.values(), None)


def test_c_cache_write_refusals(lib):
    for n in ("k", "v", "kc", "vc"):
        assert _write_c(lib, **{n: None}) == 1
    assert _write_c(lib, dtype=2) == 3
    for kw in (dict(B=0), dict(T=0), dict(N=2), dict(Hkv=0), dict(Hkv=65536), dict(d=64), dict(cu=P, cb=4), dict(cu=P, cb=2, B=1),
               dict(slots=0), dict(slots=2, idx=None), dict(sinks=-1), dict(sinks=8), dict(rows=1 << 30), dict(pb=2), dict(ib=2),
               dict(T=1 << 29)):
        assert _write_c(lib, **kw) == 2, kw
    for kw in (dict(k=P + 8), dict(vt=4), dict(kc=P + 8), dict(kcn=4), dict(vch=4), dict(pos=P + 4), dict(idx=MIS),
               dict(cu=P + 4, cb=8, B=1)):
        assert _write_c(lib, **kw) == 4, kw


def _window_step_c(lib, **kw):
    a = dict(q=P, qn=256, qh=128, k=P, kn=128, kh=128, v=P, vn=128, vh=128, pos=P, pb=8, idx=P, ib=4, kc=P, kcn=1024, kct=128, kch=128,
             vc=P, vcn=1024, vct=128, vch=128, N=3, slots=4, rows=8, H=2, Hkv=1, d=128, window=6, sinks=2, scale=0.1, dtype=1, o=P, ws=P,
             wsb=1 << 20)
    return lib.gsa_window_step(*{**a, **kw}.values(), None)


def test_c_window_step_refusals(lib):
    for n in ("q", "k", "v", "pos", "kc", "vc", "o", "ws"):
        assert _window_step_c(lib, **{n: None}) == 1
    assert _window_step_c(lib, dtype=2) == 3
    for kw in (dict(N=0), dict(N=65536), dict(slots=0), dict(slots=2, idx=None), dict(rows=7), dict(rows=1 << 30), dict(H=0), dict(Hkv=0),
               dict(H=3, Hkv=2), dict(d=64), dict(window=0), dict(sinks=-1), dict(window=1 << 30, rows=2 ** 31 - 1), dict(pb=4, ib=3),
               dict(pb=0), dict(wsb=16)):
        assert _window_step_c(lib, **kw) == 2, kw
    for kw in (dict(q=P + 8), dict(kn=4), dict(vh=4), dict(kc=P + 8), dict(vct=4), dict(pos=P + 4), dict(idx=MIS), dict(o=P + 8), dict(ws=P + 4)):
        assert _window_step_c(lib, **kw) == 4, kw


def test_c_window_step_sizes(lib):
    f = lib.gsa_window_step_workspace_bytes
    for bad in ((0, 1, 1, 1, 0, 1), (65536, 1, 1, 1, 0, 1), (1, 0, 0, 1, 0, 1), (1, 3, 2, 1, 0, 1), (1, 1, 1, 0, 0, 1), (1, 1, 1, 1, -1, 1),
                (1, 1, 1, 1 << 30, 0, 1), (1, 1, 1, 1, 0, 2)):
        assert f(*bad) == 0, bad

    def splits(N, H, Hkv, keys, dtype):          # from the parts: 130 floats a head and block
        one, n = f(N, H, Hkv, 1, 0, dtype), f(N, H, Hkv, keys, 0, dtype)
        assert (n - one) % (N * H * 130 * 4) == 0
        return max(1, (n - one) // (N * H * 130 * 4))

    assert splits(1, 16, 4, 128, 1) == 1 and splits(1, 16, 4, 129, 1) == 2 and splits(1, 16, 4, 1028, 1) == 9
    assert splits(1, 16, 4, 65536, 1) == 64 and splits(24, 16, 4, 2052, 1) == 2
    assert splits(33, 16, 4, 2052, 1) == splits(61, 16, 4, 2052, 1) == 1 and splits(33, 16, 4, 2052, 0) == 3


# ---------------------------------------------------------------------------
# What torch would lose in silence
# ---------------------------------------------------------------------------

def _calls():
    """(entry point, its floating-point arguments) of every operator."""
    lin, lstep, win, wr, st = _linear(), _linear_step(), _window(), _write(), _step()
    return [(lambda *t: linear_attention(*t[:4], initial_state=t[4]), [lin[n] for n in "qkvg"] + [Z(1, 2, D, D)]),
            (lambda *t: linear_attention_step(*t), [lstep[n] for n in "qkvg"] + [lstep["state"]]),
            (lambda *t: window_attention(*t, 3, 1), [win[n] for n in "qkv"]),
            (lambda *t: window_attention_step(*t, st["positions"], 6, 2), [st[n] for n in ("q", "k", "v", "k_cache", "v_cache")]),
            (lambda *t: window_cache_write(*t, 2), [wr[n] for n in ("k", "v", "k_cache", "v_cache")])]


@pytest.mark.parametrize("op", range(5))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_raises(op, grad):
    from torch.autograd import forward_ad as fw

    call, args = _calls()[op]
    for i in range(len(args)):
        with torch.set_grad_enabled(grad), fw.dual_level():
            dual = fw.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*args[:i], dual, *args[i + 1:])


@pytest.mark.parametrize("op", range(5))
def test_trace_raises(op):
    call, args = _calls()[op]
    with torch.no_grad(), pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, tuple(args), check_trace=False)
