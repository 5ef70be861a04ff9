"""What the gated delta rule and the RMS norm refuse, before anything is launched."""

import ctypes

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import _abi, add_rms_norm, add_rms_norm_fp8, gated_delta_rule, gated_delta_step

D, P, MIS = 128, 0x10000, 0x10002


def _rule(B=1, T=4, Hk=1, Hv=2, **kw):
    x = dict(q=torch.zeros(B, T, Hk, D), k=torch.zeros(B, T, Hk, D), v=torch.zeros(B, T, Hv, D), g=torch.zeros(B, T, Hv),
             beta=torch.zeros(B, T, Hv))
    x.update(kw)
    return x


BAD_RULE = [
    (ValueError, dict(k=torch.zeros(1, 4, 2, D))), (ValueError, dict(v=torch.zeros(1, 5, 2, D))),
    (ValueError, dict(q=torch.zeros(1, 4, 1, 64), k=torch.zeros(1, 4, 1, 64))), (ValueError, dict(v=torch.zeros(1, 4, 2, 64))),
    (ValueError, dict(q=torch.zeros(1, 4, 3, D), k=torch.zeros(1, 4, 3, D))), (ValueError, dict(g=torch.zeros(1, 4, 1))),
    (ValueError, dict(beta=torch.zeros(1, 4))), (ValueError, dict(v=torch.zeros(1, 4, 2, D, dtype=torch.bfloat16))),
    (TypeError, dict(g=torch.zeros(1, 4, 2, dtype=torch.bfloat16))), (TypeError, dict(beta=torch.zeros(1, 4, 2, dtype=torch.bfloat16))),
    (ValueError, dict(cu_seqlens=torch.tensor([0]))), (ValueError, dict(cu_seqlens=torch.tensor([0., 4.]))),
    (ValueError, dict(cu_seqlens=torch.tensor([[0, 4]]))), (ValueError, dict(initial_state=torch.zeros(2, 2, D, D))),
    (ValueError, dict(initial_state=torch.zeros(1, 2, D, D, dtype=torch.bfloat16))),
    (ValueError, dict(cu_seqlens=torch.tensor([0, 2, 4]), initial_state=torch.zeros(1, 2, D, D))),
    (RuntimeError, {}),                                              # right, but on the CPU
]


@pytest.mark.parametrize("error,kw", BAD_RULE)
def test_rule_refuses(error, kw):
    with pytest.raises(error):
        gated_delta_rule(**_rule(**kw))


def test_rule_refuses_half_and_packed_batches():
    with pytest.raises(TypeError):
        gated_delta_rule(**{n: t.half() for n, t in _rule().items() if n != "g"}, g=torch.zeros(1, 4, 2))
    with pytest.raises(ValueError, match="packed"):
        gated_delta_rule(**_rule(B=2), cu_seqlens=torch.tensor([0, 4]))


def _step(N=3, Hk=1, Hv=2, slots=4, **kw):
    x = dict(q=torch.zeros(N, Hk, D), k=torch.zeros(N, Hk, D), v=torch.zeros(N, Hv, D), g=torch.zeros(N, Hv),
             beta=torch.zeros(N, Hv), state=torch.zeros(slots, Hv, D, D))
    x.update(kw)
    return x


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(q=torch.zeros(3, D))), (ValueError, dict(g=torch.zeros(3, 1))), (ValueError, dict(state=torch.zeros(2, 2, D, D))),
    (ValueError, dict(state=torch.zeros(4, 1, D, D))), (ValueError, dict(state=torch.zeros(4, 2, D, D, dtype=torch.bfloat16))),
    (ValueError, dict(state=torch.zeros(4, 2, D, D).transpose(2, 3))), (ValueError, dict(state=torch.zeros(1, 2, D, D).expand(4, 2, D, D))),
    (ValueError, dict(state=torch.zeros(4 * 2 * D * D + 1)[1:].view(4, 2, D, D))),
    (ValueError, dict(state=torch.zeros(5 * D * D).as_strided((4, 2, D, D), (D * D, D * D, D, 1)))),
    (ValueError, dict(state=torch.zeros(9 * D * D).as_strided((4, 2, D, D), (D * D, 3 * D * D, D, 1)))),
    (ValueError, dict(state_indices=torch.zeros(2, dtype=torch.int32))), (ValueError, dict(state_indices=torch.zeros(3))),
    (RuntimeError, dict(v=torch.zeros(3, 2, D, requires_grad=True))), (RuntimeError, {})])
def test_step_refuses(error, kw):
    with pytest.raises(error):
        gated_delta_step(**_step(**kw))


def test_step_takes_states_laid_out_by_head():
    """A pool [Hv, slots] seen as [slots, Hv] passes the checks (and ends at the one for a GPU)."""
    for pool in (torch.zeros(2, 4, D, D).transpose(0, 1), torch.zeros(4, 3, D, D)[:, :2], torch.zeros(1, 2, D, D).expand(1, 2, D, D)):
        with pytest.raises(RuntimeError, match="GPU|cuda|CUDA|device"):
            gated_delta_step(**_step(N=1, slots=pool.shape[0], state=pool))


@pytest.mark.parametrize("op", [add_rms_norm, add_rms_norm_fp8])
@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(x=torch.zeros(()))), (ValueError, dict(x=torch.zeros(2, 0), weight=torch.zeros(0))),
    (ValueError, dict(x=torch.zeros(1, 32769), weight=torch.zeros(32769))), (ValueError, dict(weight=torch.zeros(7))),
    (ValueError, dict(weight=torch.zeros(8, dtype=torch.bfloat16))), (ValueError, dict(residual=torch.zeros(8))),
    (ValueError, dict(residual=torch.zeros(2, 8, dtype=torch.bfloat16))), (RuntimeError, {})])
def test_norm_refuses(op, error, kw):
    with pytest.raises(error):
        op(**{**dict(x=torch.zeros(2, 8), weight=torch.zeros(8)), **kw})


def test_norm_fp8_refuses_gradients():
    with pytest.raises(RuntimeError, match="forward only"):
        add_rms_norm_fp8(torch.zeros(2, 8, requires_grad=True), torch.zeros(8))


def test_norm_refuses_half():
    with pytest.raises(TypeError):
        add_rms_norm(torch.zeros(2, 8).half(), torch.zeros(8).half())


# ---------------------------------------------------------------------------
# The C entries: a status, nothing enqueued (the addresses are never dereferenced)
# ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    return _abi.load()


def _norm_c(lib, **kw):
    a = dict(x=P, x0=64, x1=64, res=P, r0=64, r1=64, w=P, eps=1e-6, rows=4, inner=1, D=64, dtype=1, y=P, h=P, rstd=P)
    a.update(kw)
    return lib.gsa_rms_norm(*a.values(), None)


def test_c_norm_refusals(lib):
    for n in ("x", "w", "y", "h"):
        assert _norm_c(lib, **{n: None}) == 1
    assert _norm_c(lib, dtype=2) == 3
    for kw in (dict(rows=0), dict(inner=0), dict(inner=3), dict(D=0), dict(D=32769), dict(rows=1 << 31)):
        assert _norm_c(lib, **kw) == 2
    assert _norm_c(lib, x=P + 1) == _norm_c(lib, rstd=MIS) == _norm_c(lib, dtype=0, y=MIS) == 4
    f = lib.gsa_rms_norm_fp8
    assert f(P, 64, 64, None, 0, 0, P, 1e-6, 4, 1, 64, 1, P, None, None, None) == 1
    b = lib.gsa_rms_norm_backward
    n = lib.gsa_rms_norm_backward_workspace_bytes(4, 64)
    assert n > 0 and lib.gsa_rms_norm_backward_workspace_bytes(0, 64) == lib.gsa_rms_norm_backward_workspace_bytes(4, 40000) == 0
    ok = [P, 64, 64, P, 64, 64, P, 64, 64, P, P, 4, 1, 64, 1, P, P, P, n]
    for i in (0, 3, 9, 10, 15, 16, 17):
        assert b(*(ok[:i] + [None] + ok[i + 1:]), None) == 1
    assert b(*ok[:-1], n - 1, None) == 2
    assert b(*ok[:10], MIS, *ok[11:], None) == 4


def _step_c(lib, **kw):
    a = dict(q=P, qn=128, qh=128, k=P, kn=128, kh=128, v=P, vn=256, vh=128, g=P, gn=2, gh=1, b=P, bn=2, bh=1, bt=0, idx=P, ib=4,
             S=P, sn=2 * D * D, sh=D * D, N=3, slots=4, Hk=1, Hv=2, d=128, scale=0.1, dtype=1, o=P)
    a.update(kw)
    return lib.gsa_delta_step(*a.values(), None)


def test_c_step_refusals(lib):
    for n in ("q", "k", "v", "g", "b", "S", "o"):
        assert _step_c(lib, **{n: None}) == 1
    assert _step_c(lib, dtype=5) == _step_c(lib, bt=5) == 3
    for kw in (dict(N=0), dict(N=65536), dict(slots=0), dict(Hk=0), dict(Hk=3), dict(Hv=65536), dict(d=64), dict(ib=2),
               dict(idx=None, N=5)):
        assert _step_c(lib, **kw) == 2
    for kw in (dict(S=P + 4), dict(sn=2 * D * D + 1), dict(sh=D * D + 2), dict(idx=MIS), dict(g=MIS), dict(q=P + 1), dict(o=P + 1)):
        assert _step_c(lib, **kw) == 4


def _rule_c(lib, backward=False, **kw):
    a = _abi.DeltaArgs(B=2, T=100, N=2, Hk=1, Hv=2, d=128, dtype=1, beta_dtype=0, scale=0.1)
    for n in ("q", "k", "v", "g", "beta", "o", "ws", "saved", "dout", "dq", "dk", "dv", "dg", "dbeta"):
        setattr(a, n, P)
    for n in ("q", "k", "v", "do"):
        a.__setattr__(n + "_sb", 25600), a.__setattr__(n + "_st", 256), a.__setattr__(n + "_sh", 128)
    a.ws_bytes = lib.gsa_delta_rule_workspace_bytes(2, 100, 2, 0, 1, 2, 1, int(backward))
    a.saved_bytes = lib.gsa_delta_rule_saved_bytes(2, 100, 2, 0, 1, 2, 1)
    for n, x in kw.items():
        setattr(a, n, x)
    return (lib.gsa_delta_rule_backward if backward else lib.gsa_delta_rule)(ctypes.byref(a), None)


def test_c_rule_refusals(lib):
    assert lib.gsa_delta_rule(None, None) == lib.gsa_delta_rule_backward(None, None) == 1
    for back in (False, True):
        for n in ("q", "k", "v", "g", "beta", "ws") + (("saved", "dout", "dq", "dk", "dv", "dg", "dbeta") if back else ("o",)):
            assert _rule_c(lib, back, **{n: None}) == 1, n
        assert _rule_c(lib, back, dtype=4) == _rule_c(lib, back, beta_dtype=-1) == 3
        for kw in (dict(B=0), dict(T=0), dict(N=3), dict(Hk=0), dict(Hk=3), dict(Hv=65536), dict(d=64), dict(ws_bytes=1024),
                   dict(saved_bytes=1024), dict(cu_seqlens=P, cu_bytes=4), dict(cu_seqlens=P, cu_bytes=2, B=1)):
            assert _rule_c(lib, back, **kw) == 2, kw
        for kw in (dict(q=P + 8), dict(k_st=257), dict(v_sb=4), dict(k_sh=132), dict(g=MIS), dict(beta=MIS), dict(ws=P + 8),
                   dict(state_in=P + 4), dict(cu_seqlens=P + 2, cu_bytes=4, B=1, N=2)):
            assert _rule_c(lib, back, **kw) == 4, kw
    assert _rule_c(lib, True, do_st=4) == 4


def test_c_rule_sizes(lib):
    for backward in (0, 1):
        f = lib.gsa_delta_rule_workspace_bytes
        assert f(0, 5, 1, 0, 1, 1, 1, backward) == f(1, 0, 1, 0, 1, 1, 1, backward) == f(1, 5, 1, 0, 0, 0, 1, backward) == 0
        assert f(1, 5, 1, 0, 1, 1, 7, backward) == f(1, 5, 1, 0, 2, 3, 1, backward) == 0
        assert f(1, 64, 1, 0, 2, 2, 1, backward) < f(1, 65, 1, 0, 2, 2, 1, backward)
    # what a forward keeps: a state (64 KiB) and a chunk's deltas for each chunk (64 tokens, fp32: 32) and v head
    assert lib.gsa_delta_rule_saved_bytes(1, 65, 1, 0, 2, 2, 1) == 2 * 2 * (65536 + 64 * 512)
    assert lib.gsa_delta_rule_saved_bytes(1, 65, 1, 0, 2, 2, 0) == 3 * 2 * (65536 + 32 * 512)
    # packed sequences may each leave a chunk begun: one slot more for every one of them
    assert lib.gsa_delta_rule_saved_bytes(1, 130, 5, 1, 1, 1, 1) == (2 + 5) * (65536 + 64 * 512)


def test_c_rule_sizes_at_their_ends(lib):
    """Sizes that no launch and no index holds are refused: 2**23 chunks or heads of sequences (512 threads
    each, and a launch has less than 2**32), token counts next to 2**31, products past 64 bits."""
    last = 2 ** 31 - 1
    for f in (lib.gsa_delta_rule_saved_bytes, lambda *a: lib.gsa_delta_rule_workspace_bytes(*a, 0),
              lambda *a: lib.gsa_delta_rule_workspace_bytes(*a, 1)):
        for dtype in (0, 1):
            for N in (2 ** 19 - 1, 2 ** 19):     # of 16 heads and one token each: the chunks' launches would do
                assert (f(N, 1, N, 0, 16, 16, dtype) > 0) == (f(1, 1, N, 1, 16, 16, dtype) > 0) == (N < 2 ** 19)
            for packed in (0, 1):
                assert f(1, last, 1, packed, 1, 1, dtype) == f(1, last, 1, packed, last, last, dtype) == 0
            assert f(last, last, last, 0, last, last, dtype) == f(2 ** 29, 64, 2 ** 29, 0, 32, 32, dtype) == 0
    assert lib.gsa_delta_rule_saved_bytes(1, 64 * 2 ** 23, 1, 0, 1, 1, 1) > 0 == lib.gsa_delta_rule_saved_bytes(1, 64 * 2 ** 23 + 1, 1, 0, 1, 1, 1)


def test_c_rule_shape(lib):
    """0 with the byte counts; half heads for few of them, whole ones alone and two on a CU for many; segments for long rows."""
    f = lib.gsa_delta_rule_shape
    assert f(1, 5, 1, 0, 2, 3, 1) == f(0, 5, 0, 0, 1, 1, 1) == f(1, 5, 1, 0, 1, 1, 7) == f(1, 2 ** 31 - 1, 1, 0, 1, 1, 1) == 0
    for dtype in (0, 1):
        assert [f(B, 100, B, 0, 16, 16, dtype) for B in (1, 8, 9, 16, 17, 40)] == [1, 1, 2, 2, 3, 3]
        assert [f(1, 100 * N, N, 1, 16, 16, dtype) for N in (1, 9, 32, 33, 100)] == [1, 1, 1, 2, 2]
        assert f(1, 16384, 1, 0, 16, 16, dtype) == 6


# ---------------------------------------------------------------------------
# What torch would lose in silence
# ---------------------------------------------------------------------------

def _calls():
    """(entry point, its floating-point arguments) of every operator."""
    names = ("q", "k", "v", "g", "beta")
    rule, step, x = _rule(), _step(), torch.ones(2, 8)
    return [(lambda *t: gated_delta_rule(*t[:5], initial_state=t[5]), [rule[n] for n in names] + [torch.zeros(1, 2, D, D)]),
            (lambda *t: gated_delta_step(*t), [step[n] for n in names] + [step["state"]]),
            (lambda *t: add_rms_norm(t[0], t[1], residual=t[2]), [x, torch.ones(8), x.clone()]),
            (lambda *t: add_rms_norm_fp8(t[0], t[1], residual=t[2]), [x, torch.ones(8), x.clone()])]


@pytest.mark.parametrize("op", range(4))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_raises(op, grad):
    """A dual tensor needs no gradient, and its data is there: the result would come without its tangent."""
    from torch.autograd import forward_ad as fw

    call, args = _calls()[op]
    for i in range(len(args)):
        with torch.set_grad_enabled(grad), fw.dual_level():
            dual = fw.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*args[:i], dual, *args[i + 1:])
    with fw.dual_level(), pytest.raises(RuntimeError, match="GPU|CUDA|device"):
        call(*args)                              # no tangent among them: on to the next check


def test_forward_mode_over_the_backward_pass_raises():
    from torch.autograd import forward_ad as fw

    from gsa_gdn_benchmarkstudy_amd.delta import _once

    class Double(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return 2 * x

        @_once
        def backward(ctx, dy):
            return 2 * dy

    x = torch.ones(3, requires_grad=True)
    with fw.dual_level():
        dy = fw.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(Double.apply(x), x, dy)


@pytest.mark.parametrize("op", range(4))
def test_trace_raises(op):
    call, args = _calls()[op]
    with torch.no_grad(), pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, tuple(args), check_trace=False)
