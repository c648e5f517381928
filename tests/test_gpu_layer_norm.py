"""ops.layer_norm against the formula in 64 bits, forward and gradients.

Bounds are derived.  u = 2^-24, b = 2^-8 for bf16 outputs (else 0), D the row's length; a sum
over a row is a chain of at most c = 20 + D / 256 fp32 additions per thread and tree, so
it is off by c u sum|.|.  With A = mean|x| r (mean error in units of the deviation):
  xh is off by e = (c A + (c + 6) |xh|) u   (mean; variance, root, product)
  y  by |w| e + 2 u |y| + b |y|
  dx = r (g - mean(g) - xh mean(g xh)), M = mean|g|, N = mean|g xh|: each mean is off by
       c u of its absolute mean and by what xh is off, so dx by
       r (4 u |g| + c u M + |xh| (c u N + mean(|g| e)) + e N) + 8 u |dx| + b |dx|
  dw, db: a chain of rows / 16,384 + 50 additions at most (a team's rows, then fixed trees):
       (rows / 16,384 + 52) u sum|dy xh| + sum(|dy| e)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def reference(x, w, b, eps, dy):
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else 0.0
    whalf = 2.0 ** -8 if (w if w is not None else b) is not None and (w if w is not None else b).dtype == torch.bfloat16 else 0.0
    D = x.shape[-1]
    x, dy = x.detach().double().reshape(-1, D), dy.double().reshape(-1, D)
    ww = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    bb = torch.zeros_like(ww) if b is None else b.detach().double()
    c = 20 + D / 256
    mu = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((x - mu).square().mean(1, keepdim=True) + eps)
    xh = (x - mu) * r
    e = (c * x.abs().mean(1, keepdim=True) * r + (c + 6) * xh.abs()) * U
    y = xh * ww + bb
    g = dy * ww
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    dx = r * (g - mean(g) - xh * mean(g * xh))
    edx = r * (4 * U * g.abs() + c * U * mean(g.abs()) + xh.abs() * (c * U * mean((g * xh).abs()) + mean(g.abs() * e))
               + e * mean((g * xh).abs()))
    chain = x.shape[0] / 16384 + 52
    dw, db = (dy * xh).sum(0), dy.sum(0)
    return ((y, ww.abs() * e + 2 * U * (y.abs() + bb.abs()) + half * y.abs()), (dx, edx + (8 * U + half) * dx.abs()),
            (dw, chain * U * (dy * xh).abs().sum(0) + (dy.abs() * e).sum(0) + whalf * dw.abs()),
            (db, chain * U * dy.abs().sum(0) + whalf * db.abs()))


def check(x, w, b, eps=1e-6):
    from mygenerativerecommenders_amd import ops
    g = torch.Generator(device="cuda").manual_seed(x.shape[-1])
    dy = torch.randn(x.shape, device="cuda", generator=g).to(x.dtype)
    x, w, b = (t if t is None else t.detach().requires_grad_(True) for t in (x, w, b))
    y = ops.layer_norm(x, w, b, eps)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = iter(torch.autograd.grad(y, leaves, dy))
    got = [y.detach()] + [None if t is None else next(grads) for t in (x, w, b)]
    for name, t, s, (ref, lim) in zip(("y", "dx", "dw", "db"), got, (x, x, w, b), reference(x, w, b, eps, dy)):
        if t is None:
            continue
        assert t.dtype == s.dtype and t.shape == s.shape, name
        assert torch.isfinite(t).all(), name
        worst = ((t.double().reshape(ref.shape) - ref).abs() / (lim + 1e-30)).max().item() if t.numel() else 0.0
        assert worst <= 1.0, (name, worst)
    return got


def inputs(rows, D, dtype, wdtype=None, seed=0, wide=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + D)
    x = (2 * torch.randn(rows, D + wide, device="cuda", generator=g) + 0.5).to(dtype)[:, :D]
    if wdtype is None:
        return x, None, None
    return (x, (1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(wdtype),
            torch.randn(D, device="cuda", generator=g).to(wdtype))


DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


# every team and vector count, the border of each, and the looping kernels
@DTYPES
@pytest.mark.parametrize("D", [1, 2, 3, 8, 31, 50, 64, 65, 128, 200, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2048,
                               2049, 4095, 4096, 4097, 8192, 8193, 16384, 20000])
def test_widths(D, dtype):
    check(*inputs(37, D, dtype, torch.float32))


@DTYPES
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 1000, 40003])
def test_rows(rows, dtype):
    check(*inputs(rows, 50, dtype, torch.float32, wide=14))


@DTYPES
def test_without_weight(dtype):
    check(*inputs(300, 256, dtype))


@DTYPES
def test_weight_alone_and_bias_alone(dtype):
    x, w, b = inputs(70, 96, dtype, torch.float32)
    check(x, w, None)
    check(x, None, b)


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)])
def test_bf16_weights(dtype, wdtype):
    check(*inputs(129, 320, dtype, wdtype))


def test_many_rows_of_a_wide_row():
    check(*inputs(3001, 4096, torch.bfloat16, torch.float32))


@DTYPES
def test_strides(dtype):
    from mygenerativerecommenders_amd import ops
    x, w, b = inputs(60, 50, dtype, torch.float32)
    want = ops.layer_norm(x, w, b)
    shapes = [torch.cat([torch.ones_like(x[:, :1]), x], 1)[:, 1:],  # odd row stride, odd first element
              torch.cat([x, x], 1)[:, 50:], x.t().contiguous().t(),  # columns apart
              torch.stack([x, x], 1)[:, 0]]
    for t in shapes:
        assert torch.equal(ops.layer_norm(t, w, b), want)
    three = x.view(3, 20, 50).transpose(0, 1)  # rows without one stride
    assert torch.equal(ops.layer_norm(three, w, b), want.view(3, 20, 50).transpose(0, 1))
    assert torch.equal(ops.layer_norm(x[:1].expand(60, 50), w, b), want[:1].expand(60, 50))
    check(three, w, b)
    check(x[:1].expand(60, 50), w, b)
    assert ops.layer_norm(x[0], w, b).shape == (50,)


def test_expanded_output_gradient():
    """sum().backward() hands the backward a gradient without strides."""
    from mygenerativerecommenders_amd import ops
    x, w, b = (t.requires_grad_(True) for t in inputs(40, 50, torch.float32, torch.float32))
    ops.layer_norm(x, w, b).sum().backward()
    ref = reference(x, w, b, 1e-6, torch.ones(40, 50, device="cuda"))
    for t, (y, lim) in zip((x, w, b), ref[1:]):
        assert ((t.grad.double() - y).abs() <= lim + 1e-30).all()


def test_far_means_and_constant_rows():
    """A mean a thousand deviations away, a constant row (variance 0: eps alone), a tiny row."""
    x, w, b = inputs(64, 256, torch.float32, torch.float32)
    x = x.clone()
    x[:16] += 2000
    x[16:20] = 3.25
    x[20:24] *= 1e-6
    check(x, w, b)


def test_each_wanted_gradient_alone():
    from mygenerativerecommenders_amd import ops
    x, w, b = inputs(90, 200, torch.float32, torch.float32)
    dy = torch.randn_like(x)
    every = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(ops.layer_norm(*every), every, dy)
    for i in range(3):
        args = [x, w, b]
        args[i] = args[i].clone().requires_grad_(True)
        (g,) = torch.autograd.grad(ops.layer_norm(*args), args[i], dy)
        assert torch.equal(g, want[i])


def test_not_finite_rows_stay_alone():
    from mygenerativerecommenders_amd import ops
    x, w, b = inputs(40, 50, torch.float32, torch.float32)
    want = ops.layer_norm(x, w, b)
    x = x.clone()
    x[7, 3], x[20, 49] = float("nan"), float("inf")
    got = ops.layer_norm(x, w, b)
    rest = [i for i in range(40) if i not in (7, 20)]
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[[7, 20]]).all()


def test_rows_beyond_32_bits():
    from mygenerativerecommenders_amd import ops
    x, w, b = inputs(9, 64, torch.bfloat16, torch.float32)
    big = torch.empty(60000 * 40000, dtype=torch.bfloat16, device="cuda").view(60000, 40000)
    far = big[-9:, -64:]
    far.copy_(x)
    assert torch.equal(ops.layer_norm(far, w, b), ops.layer_norm(x, w, b))
    every = big[:, :64]
    every.zero_()
    every[-9:] = x
    assert torch.equal(ops.layer_norm(every, w, b)[-9:], ops.layer_norm(x, w, b))


def test_second_derivative():
    """create_graph: the gradient of a gradient, against torch's own on the same values.
    Both are fp32 chains of some tens of operations over rows of 24 values of order one."""
    from mygenerativerecommenders_amd import ops
    outs = []
    for f in (ops.layer_norm, lambda x, w, b: torch.nn.functional.layer_norm(x, (24,), w, b, 1e-6)):
        x, w, b = (t.clone().requires_grad_(True) for t in inputs(10, 24, torch.float32, torch.float32))
        (g,) = torch.autograd.grad((f(x, w, b) ** 3).sum(), x, create_graph=True)
        outs.append(torch.autograd.grad((g ** 2).sum(), (x, w, b)))
    for p, q in zip(*outs):
        assert (p - q).abs().max() <= 2e-4 * (1 + q.abs().max())


def test_same_bits_every_run_on_another_stream_and_captured():
    from mygenerativerecommenders_amd import ops
    x, w, b = (t.requires_grad_(True) for t in inputs(5000, 256, torch.bfloat16, torch.float32))
    dy = torch.randn_like(x)

    def run():
        y = ops.layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(3):
        with torch.no_grad():
            dy.mul_(-1.5)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(outs, run())), i


def test_postprocessor_runs_it():
    from mygenerativerecommenders_amd import _lib
    from mygenerativerecommenders_amd.postprocessors import LayerNormEmbeddingPostprocessor
    m = LayerNormEmbeddingPostprocessor(50)
    x = torch.randn(4, 33, 64, device="cuda", requires_grad=True)
    _lib.timing_enable(True)
    try:
        _lib.kernel_times()
        y = m(x)
        y.square().sum().backward()
        t = _lib.kernel_times(("layer_norm_fwd", "layer_norm_bwd"))
    finally:
        _lib.timing_enable(False)
    assert t["layer_norm_fwd"][1] == 1 and t["layer_norm_bwd"][1] == 1
    z = x.detach().cpu().requires_grad_(True)
    ref = m(z)  # the CPU keeps torch's
    ref.square().sum().backward()
    assert torch.allclose(y.detach().cpu(), ref, rtol=1e-5, atol=1e-5)
    assert torch.allclose(x.grad.cpu(), z.grad, rtol=1e-4, atol=1e-4)
    assert (x.grad[..., 50:] == 0).all()
    assert m(x.double()).dtype == torch.float64 and m(x.half()).dtype == torch.float16
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert m(x.bfloat16()).dtype == torch.float32
    with pytest.raises(RuntimeError):
        m(x[..., :20])


def test_refusals_and_empty():
    from mygenerativerecommenders_amd import _lib, ops
    x, w, b = inputs(4, 16, torch.float32, torch.float32)
    with pytest.raises(_lib.GrError, match="CPU tensor"):
        ops.layer_norm(x.cpu())
    for bad in (x.half(), x.double(), x.long()):
        with pytest.raises(TypeError):
            ops.layer_norm(bad)
    with pytest.raises(TypeError):
        ops.layer_norm(x, w, b.bfloat16())
    with pytest.raises(TypeError):
        ops.layer_norm(x, w.half())
    for bad in (w[:8], w[None]):
        with pytest.raises(ValueError):
            ops.layer_norm(x, bad)
    for bad in (x[:, :0], x[0, 0]):
        with pytest.raises(ValueError):
            ops.layer_norm(bad)
    e, w2, b2 = (t.detach().requires_grad_(True) for t in (x[:0], w, b))
    ops.layer_norm(e, w2, b2).sum().backward()
    assert e.grad.shape == (0, 16) and (w2.grad == 0).all() and (b2.grad == 0).all()


def test_no_derivative_is_dropped_in_silence():
    """Forward-mode derivatives and traces, which the kernels know nothing of, raise; a batched map runs
    them in a loop, a compiled function around them."""
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx
    from mygenerativerecommenders_amd import ops
    x, w, b = inputs(6, 16, torch.float32, torch.float32)
    for grad in (False, True):
        with fw.dual_level():
            for i, t in enumerate((x, w, b)):
                args = [x, w, b]
                args[i] = fw.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    ops.layer_norm(*args)
    f = lambda t: ops.layer_norm(t, w, b)  # noqa: E731
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(f)(x)
    with pytest.raises(NotImplementedError, match="plain tensors"):
        torch.func.grad(lambda t: f(t).sum())(x)
    assert torch.equal(torch.func.vmap(f)(torch.stack([x, 2 * x])), torch.stack([f(x), f(2 * x)]))
    assert torch.equal(torch.compile(f, backend="eager")(x), f(x))


def test_postprocessor_keeps_the_forward_mode_derivative():
    import torch.autograd.forward_ad as fw
    from mygenerativerecommenders_amd.postprocessors import LayerNormEmbeddingPostprocessor
    x, way = torch.randn(2, 6, 16, device="cuda")
    m = LayerNormEmbeddingPostprocessor(12)
    norm = lambda t: torch.nn.functional.layer_norm(t[..., :12], (12,), eps=1e-6)  # noqa: E731
    for grad in (False, True):
        with fw.dual_level():
            dual = fw.make_dual(x.clone().requires_grad_(grad), way)
            got, want = (fw.unpack_dual(f(dual)).tangent for f in (m, norm))
            assert want is not None and torch.equal(got, want)
    leaf = x.clone().requires_grad_(True)
    name = m(leaf).grad_fn.name()
    assert "LayerNorm" in name and "Native" not in name


def test_postprocessor_traces_to_torchs_norm():
    """Every tracer sees torch's layer norm, and what it made runs without this package's operators."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from mygenerativerecommenders_amd.postprocessors import LayerNormEmbeddingPostprocessor
    x, other = torch.randn(2, 6, 16, device="cuda")
    m = LayerNormEmbeddingPostprocessor(12)
    norm = lambda t: torch.nn.functional.layer_norm(t[..., :12], (12,), eps=1e-6)  # noqa: E731
    traced = [make_fx(m)(x), make_fx(m, tracing_mode="fake")(x), make_fx(m, pre_dispatch=True)(x),
              torch.jit.trace(m, x), torch.fx.symbolic_trace(m),
              torch.jit.script(m), torch.export.export(m, (x,)).module(), torch.compile(m, backend="eager")]
    for t in traced:
        assert torch.equal(t(other), norm(other))
    assert all("layer_norm" in t.code and "gr_amd" not in t.code for t in traced[:-1])
    assert torch.allclose(torch.func.vmap(m)(torch.stack([x, other])), torch.stack([norm(x), norm(other)]), atol=1e-5)


@DTYPES
def test_overlapping_rows(dtype):
    """Rows that share columns with the next (a window moved by less than a row)."""
    from mygenerativerecommenders_amd.postprocessors import LayerNormEmbeddingPostprocessor
    g = torch.Generator(device="cuda").manual_seed(3)
    line = torch.randn(400, device="cuda", generator=g).to(dtype)
    _, w, b = inputs(2, 50, dtype, torch.float32)
    for step in (1, 7, 49):
        x = line.unfold(0, 50, step)
        assert x.stride() == (step, 1)
        check(x, w, b)
        y = LayerNormEmbeddingPostprocessor(50)(x)
        (ref, lim), *_ = reference(x, None, None, 1e-6, torch.zeros_like(x))
        assert ((y.double() - ref).abs() <= lim + 1e-30).all()


def test_refuses_rows_that_32_bits_do_not_count():
    """A width of 2^32 + 50 is not one of 50; the rows are one element, expanded."""
    from mygenerativerecommenders_amd import ops
    for d in (1 << 29, (1 << 32) + 50):
        with pytest.raises(ValueError, match="2\\^29"):
            ops.layer_norm(torch.zeros(1, 1, device="cuda").expand(2, d))
