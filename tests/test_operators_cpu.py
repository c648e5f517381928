"""What the attention, layer norm and 8-bit AdamW entries refuse, without a GPU: the checks run
before any HIP call."""
import ctypes

import pytest
import torch

from mygenerativerecommenders_amd import _lib, ops
from mygenerativerecommenders_amd.optim import FlatAdamW

P = 4096  # a pointer that is never followed: each call below is refused


def attn(**kw):
    a = dict(q=P, ld_q=8, hs_q=8, k=P, ld_k=8, hs_k=8, v=P, ld_v=8, hs_v=8, offsets=P, B=1, rows=4, H=2, Hkv=1, d=8, dv=8,
             causal=1, scale=1.0, bf16=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(offsets=None), dict(B=-1), dict(rows=-1),
                                 dict(H=0), dict(Hkv=0), dict(H=3, Hkv=2), dict(d=3), dict(d=7, bf16=1), dict(d=257), dict(dv=0), dict(dv=300),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(q=P + 2), dict(ld_k=-8), dict(ld_v=1 << 22), dict(ld_q=9, bf16=1), dict(hs_k=9, bf16=1),
                                 dict(d=9, bf16=1), dict(H=1 << 15, Hkv=1 << 15, dv=128),
                                 dict(rows=1 << 31), dict(rows=1 << 30, H=4096, Hkv=4096)], ids=str)
def test_attention_refuses(bad):
    with pytest.raises(_lib.GrError, match="gr_jagged_attn_fwd"):
        _lib.call("gr_jagged_attn_fwd", *attn(**bad), P, None, None, None)
    with pytest.raises(_lib.GrError, match="gr_jagged_attn_bwd"):
        _lib.call("gr_jagged_attn_bwd", *attn(**bad), P, P, P, P, P, P, P, P, 1 << 40, None)


def test_attention_backward_refuses_missing_buffers():
    for i in range(8):
        bufs = [P] * 8
        bufs[i] = None
        with pytest.raises(_lib.GrError):
            _lib.call("gr_jagged_attn_bwd", *attn(bf16=1), *bufs, 1 << 20, None)
    n = _lib.lib().gr_jagged_attn_bwd_workspace_size(4, 2)
    assert n == 32
    with pytest.raises(_lib.GrError, match="workspace"):
        _lib.call("gr_jagged_attn_bwd", *attn(), *[P] * 8, n - 1, None)
    with pytest.raises(_lib.GrError):
        _lib.call("gr_jagged_attn_fwd", *attn(), None, None, None, None)


def test_layer_norm_refuses():
    ok = dict(x=P, ld_x=8, rows=4, D=8, w=None, b=None, types=0, eps=1e-6, y=P, ld_y=8, stats=None, stream=None)
    for bad in (dict(x=None), dict(y=None), dict(rows=-1), dict(D=0), dict(types=4), dict(types=-1), dict(ld_x=7),
                dict(ld_x=-8), dict(ld_y=7), dict(ld_y=0)):
        with pytest.raises(_lib.GrError, match="gr_layer_norm_fwd"):
            _lib.call("gr_layer_norm_fwd", *dict(ok, **bad).values())
    ok = dict(dy=P, ld_dy=8, x=P, ld_x=8, rows=4, D=8, w=None, types=0, stats=P, dx=P, ld_dx=8, dw=None, db=None, ws=None,
              n=0, stream=None)
    for bad in (dict(dy=None), dict(x=None), dict(stats=None), dict(rows=-1), dict(D=0), dict(types=4), dict(ld_dy=7),
                dict(ld_x=7), dict(ld_dx=7), dict(dw=P), dict(db=P), dict(dw=P, ws=P, n=8)):
        with pytest.raises(_lib.GrError, match="gr_layer_norm_bwd"):
            _lib.call("gr_layer_norm_bwd", *dict(ok, **bad).values())
    assert _lib.lib().gr_layer_norm_bwd_workspace_size(4, 8, 0) >= 2 * 8 * 4
    assert _lib.lib().gr_layer_norm_bwd_workspace_size(0, 8, 0) == 0
    _lib.call("gr_layer_norm_fwd", None, 8, 0, 8, None, None, 0, 1e-6, None, 8, None, None)


def test_adamw8_refuses():
    u64, i64 = ctypes.c_uint64 * 1, ctypes.c_int64 * 1
    hyper = (1e-3, 0.9, 0.999, 1e-8, 0.0, None)

    def call(params=P, grads=P, off=0, numel=8, n=1, bufs=(P,) * 6):
        lists = [ctypes.addressof(a) for a in (pp, gg, oo, nn)] if n else [None] * 4
        pp[0], gg[0], oo[0], nn[0] = params, grads, off, numel
        _lib.call("gr_adamw8_step", *lists, n, *bufs, *hyper)

    pp, gg, oo, nn = u64(), u64(), i64(), i64()
    for bad in (dict(params=0), dict(grads=0), dict(off=-64), dict(off=32), dict(numel=-1), dict(n=-1),
                *(dict(bufs=(P,) * i + (None,) + (P,) * (5 - i)) for i in range(6)), dict(bufs=(P + 1,) + (P,) * 5)):
        with pytest.raises(_lib.GrError, match="gr_adamw8_step"):
            call(**bad)
    call(n=0, bufs=(None,) * 6)
    call(numel=0)  # nothing to do


def test_python_entries_refuse_cpu_tensors():
    x = torch.zeros(3, 2, 8)
    with pytest.raises(_lib.GrError, match="CPU tensor"):
        ops.jagged_attention(x, x, x, torch.tensor([0, 3]))
    with pytest.raises(_lib.GrError, match="CPU tensor"):
        ops.layer_norm(x)
    p = torch.nn.Parameter(torch.zeros(8))
    for bits in (0, 4, 16):
        with pytest.raises(ValueError, match="state_bits"):
            FlatAdamW([p], state_bits=bits)
    p.grad = torch.zeros(8)
    with pytest.raises(TypeError):
        FlatAdamW([p], state_bits=8).step()


def test_layer_norm_postprocessor_on_the_cpu_is_torchs():
    from mygenerativerecommenders_amd.postprocessors import LayerNormEmbeddingPostprocessor
    x = torch.randn(5, 7, 64, dtype=torch.float64, requires_grad=True)
    y = LayerNormEmbeddingPostprocessor(50)(x)
    assert torch.equal(y, torch.nn.functional.layer_norm(x[..., :50], (50,), eps=1e-6))
    assert torch.autograd.gradcheck(LayerNormEmbeddingPostprocessor(6), (x[0, :2, :8].detach().requires_grad_(True),))


def test_attention_backward_refuses_queries_that_share_elements():
    """The key rows' pass takes rows past a sequence's end as zeros, which such rows are not."""
    for ld in (0, 4):
        with pytest.raises(_lib.GrError, match="query rows"):
            _lib.call("gr_jagged_attn_bwd", *attn(ld_q=ld), *[P] * 8, 1 << 20, None)


def test_operators_refuse_what_they_would_drop():
    """Tangents and traces, before anything of the GPU's is asked."""
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx
    x, q, offsets = torch.randn(3, 8), torch.randn(3, 2, 8), torch.tensor([0, 3])
    norm = lambda t: _lib.nodes().layer_norm.default(t, None, None, 1e-6)  # noqa: E731
    attend = lambda t: _lib.nodes().jagged_attention.default(t, t, t, offsets, True, 1.0)  # noqa: E731
    for f, t in ((norm, x), (attend, q)):
        with fw.dual_level():
            for grad in (False, True):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(fw.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t)))
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(f)(t)
        with pytest.raises(NotImplementedError):
            make_fx(f, tracing_mode="fake")(t)
        with pytest.raises(NotImplementedError):
            torch.func.jvp(f, (t,), (t,))


def test_layer_norm_postprocessor_can_be_traced_and_scripted():
    """Symbolic proxies and TorchScript reach torch's norm as they do without a kernel."""
    from mygenerativerecommenders_amd.postprocessors import LayerNormEmbeddingPostprocessor
    m, x = LayerNormEmbeddingPostprocessor(5), torch.randn(4, 8)
    want = torch.nn.functional.layer_norm(x[..., :5], (5,), eps=1e-6)
    for t in (torch.fx.symbolic_trace(m), torch.jit.script(m), torch.jit.trace(m, x)):
        assert torch.equal(t(x), want) and "layer_norm" in t.code


def test_a_trace_that_makes_the_first_call_holds_no_addresses():
    """In a process of its own, as a process loads the operators once."""
    import subprocess
    import sys
    code = ("import torch; from torch.fx.experimental.proxy_tensor import make_fx\n"
            "from mygenerativerecommenders_amd import _lib\n"
            "g = make_fx(lambda x: (_lib.nodes(), x + 1)[1], pre_dispatch=True)(torch.zeros(3))\n"
            "assert 'gr_amd' not in g.code, g.code\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120)


def test_the_operators_alone_raise():
    """A process that loads libgr_torch.so by itself (for a saved trace, say) has no kernels behind it."""
    import subprocess
    import sys
    code = (f"import torch; torch.ops.load_library({_lib.NODES_PATH!r})\n"
            "try:\n    torch.ops.gr_amd.layer_norm(torch.zeros(2, 8), None, None, 1e-6)\n"
            "except RuntimeError as e:\n    assert '_lib.nodes()' in str(e), e\n"
            "else:\n    raise SystemExit(1)\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120)


@pytest.mark.parametrize("D", [1 << 29, (1 << 31) - 1])
def test_layer_norm_refuses_rows_that_32_bits_do_not_count(D):
    with pytest.raises(_lib.GrError, match="gr_layer_norm_fwd"):
        _lib.call("gr_layer_norm_fwd", P, D, 1, D, None, None, 0, 1e-6, P, D, None, None)
    with pytest.raises(_lib.GrError, match="gr_layer_norm_bwd: bad args"):
        _lib.call("gr_layer_norm_bwd", P, D, P, D, 1, D, None, 0, P, P, D, None, None, None, 0, None)


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_state_loaded_on_the_cpu(bits):
    """It waits there as it was saved, a copy of its own, and a refused one leaves it."""
    def moments(p, step):
        st = {"step": torch.tensor(float(step)), "exp_avg": torch.ones_like(p), "exp_avg_sq": torch.ones_like(p)}
        blocks = -(-p.numel() // 64)
        return dict(st, exp_avg_scale=torch.ones(blocks), exp_avg_sq_scale=torch.ones(blocks)) if bits == 8 else st

    params = [torch.nn.Parameter(torch.zeros(n)) for n in (7, 70)]
    opt = FlatAdamW(params, state_bits=bits)
    saved = dict(opt.state_dict(), state={i: moments(p.detach(), 3) for i, p in enumerate(params)})
    opt.load_state_dict(saved)
    saved["state"][1]["step"] += 1
    with pytest.raises(ValueError, match="steps"):
        opt.load_state_dict(saved)
    assert [float(opt.state[p]["step"]) for p in params] == [3, 3]
    assert all((opt.state[p]["exp_avg"].float() == 1).all() for p in params)
