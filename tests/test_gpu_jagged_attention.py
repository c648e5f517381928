"""ops.jagged_attention against the formula in 64 bits, forward and gradients.

Bounds are derived, not fitted.  With u = 2^-24 (half a step of fp32) and b = 2^-8 (half a
step of bf16; 0 where the operands are fp32):
  * a score is a sum of d products: error at most (d + 2) u scale sum|q k| =: e, which is the
    relative error of its probability, as is the log-sum's (the largest e of the row) and that
    of the exponential and its argument, (2 + |score|) u.  So P is off by at most
    r P, r = e + max e + (8 + n + 2 max|score|) u, n terms in its sum;
  * a product with P (rounded to bf16: b P) over n rows is off by (r + b + n u) P|x|;
  * D = sum(dO O) is off by b dO|O| (O is held in the operands' type) + what O is off by times
    |dO| + dv u dO|O|, dP by dv u |dO||V|, so dS by r |dS| + P (those two);
  * the result is rounded once more to its type: b of itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def reference(q, k, v, offsets, causal, scale, dout):
    """(out, dq, dk, dv) in 64 bits and the bound of each, from the inputs' own values."""
    b = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    q, k, v, dout = (t.detach().double() for t in (q, k, v, dout))
    H, group, d, w = q.shape[1], q.shape[1] // k.shape[1], q.shape[2], v.shape[2]
    res = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (dout, q, k, v)]
    lim = [torch.zeros_like(t) for t in res]
    ends = offsets.tolist()
    for s, e in zip(ends, ends[1:]):
        n = e - s
        for h in range(H if n else 0):
            j = h // group
            Q, K, V, G = q[s:e, h], k[s:e, j], v[s:e, j], dout[s:e, h]
            S = scale * (Q @ K.T)
            live = torch.ones(n, n, dtype=torch.bool, device=q.device)
            if causal:
                live = live.tril()
            err = (d + 2) * U * scale * (Q.abs() @ K.abs().T) * live
            S = S.masked_fill(~live, -math.inf)
            P = torch.softmax(S, -1)
            r = err + err.amax(1, keepdim=True) + (8 + n + 2 * (S.abs() * live).nan_to_num(0, 0, 0).amax(1, keepdim=True)) * U
            O = P @ V
            eO = (P * (r + b + n * U)) @ V.abs()
            dP = G @ V.T
            D = (G * O).sum(1, keepdim=True)
            eD = ((b + w * U) * (G * O).abs() + G.abs() * eO).sum(1, keepdim=True)
            dS = P * (dP - D)
            eS = r * dS.abs() + P * (eD + w * U * (G.abs() @ V.abs().T)) + (b + n * U) * dS.abs()
            parts = [(O, eO), (scale * (dS @ K), scale * (eS @ K.abs())), (scale * (dS.T @ Q), scale * (eS.T @ Q.abs())),
                     (P.T @ G, (P * (r + b + n * U)).T @ G.abs())]
            for i, (at, (x, ex)) in enumerate(zip((h, h, j, j), parts)):
                res[i][s:e, at] += x
                lim[i][s:e, at] += ex
    return res, [t + (b + 4 * U) * x.abs() + 1e-30 for t, x in zip(lim, res)]


def make(lengths, H, Hkv, d, dv, dtype, spare=0, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(lengths) + d)
    offsets = torch.tensor([0] + list(lengths)).cumsum(0).cuda()
    rows = int(offsets[-1]) + spare
    wide = torch.randn(rows, H * d + Hkv * (d + dv), device="cuda", generator=g).to(dtype)
    q = (spread * wide[:, :H * d]).to(dtype).view(rows, H, d)
    k = wide[:, H * d:(H + Hkv) * d].view(rows, Hkv, d)
    v = wide[:, (H + Hkv) * d:].view(rows, Hkv, dv)
    dout = torch.randn(rows, H, dv, device="cuda", generator=g).to(dtype)
    return q, k, v, offsets, dout


def run(q, k, v, offsets, dout, **kw):
    from mygenerativerecommenders_amd import ops
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = ops.jagged_attention(q, k, v, offsets, **kw)
    return [out.detach(), *torch.autograd.grad(out, (q, k, v), dout)]


def check(q, k, v, offsets, dout, causal=True, scale=None):
    got = run(q, k, v, offsets, dout, causal=causal, **({} if scale is None else {"scale": scale}))
    ref, lim = reference(q, k, v, offsets, causal, q.shape[2] ** -0.5 if scale is None else scale, dout)
    for name, x, y, e in zip(("out", "dq", "dk", "dv"), got, ref, lim):
        assert x.dtype == q.dtype and x.shape == y.shape
        assert torch.isfinite(x).all(), name
        worst = ((x.double() - y).abs() / e).max().item() if x.numel() else 0.0
        assert worst <= 1.0, (name, worst)
    return got


DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


@DTYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("lengths", [[1], [0, 1, 2, 0, 3], [31, 32, 33], [127, 128, 129, 0], [64, 65, 300, 7, 211]],
                         ids=str)
def test_lengths(lengths, causal, dtype):
    check(*make(lengths, 2, 2, 50, 50, dtype), causal=causal)


@DTYPES
@pytest.mark.parametrize("d,dv", [(1, 1), (3, 5), (7, 4), (8, 8), (33, 50), (50, 33), (64, 64), (65, 64), (100, 96),
                                  (128, 128), (129, 40), (40, 200), (255, 256), (256, 256)])
def test_widths(d, dv, dtype):
    check(*make([37, 130, 1], 2, 1, d, dv, dtype))


@DTYPES
@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 3), (4, 1), (6, 2), (8, 8)])
def test_shared_heads(H, Hkv, dtype):
    check(*make([150, 33, 0, 70], H, Hkv, 64, 64, dtype))


@DTYPES
@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_rows(d, dtype):
    check(*make([1111, 2059], 1, 1, d, d, dtype), causal=d != 128)


@DTYPES
def test_many_short_sequences(dtype):
    lengths = [(7 * i) % 12 for i in range(700)]
    check(*make(lengths, 2, 1, 16, 24, dtype))


@DTYPES
@pytest.mark.parametrize("d", [62, 128, 256])
def test_more_tiles_than_the_chip_holds(d, dtype):
    check(*make([300] + [(37 * i) % 150 for i in range(240)], 4, 2, d, d, dtype))


@DTYPES
@pytest.mark.parametrize("d", [50, 256])
def test_rows_of_no_sequence_are_zero_and_never_read(d, dtype):
    q, k, v, offsets, dout = make([40, 0, 129], 2, 1, d, d, dtype, spare=300)
    n = int(offsets[-1])
    want = run(q[:n], k[:n], v[:n], offsets, dout[:n])
    q, k, v, dout = (t.clone() for t in (q, k, v, dout))
    for t in (q, k, v, dout):
        t[n:] = float("nan")
    for x, y in zip(run(q, k, v, offsets, dout), want):
        assert torch.equal(x[:n], y) and (x[n:] == 0).all()


@DTYPES
@pytest.mark.parametrize("many", [0, 400])
def test_some_sequences_of_a_batch(many, dtype):
    """A slice of the offsets: the rows before its first sequence are of no sequence either."""
    lengths = [140, 33] + [50, 0, 129] + [1] * many + [70]
    q, k, v, offsets, dout = make(lengths, 2, 1, 40, 40, dtype)
    ends = offsets[2:6 + many]
    lo, hi = int(ends[0]), int(ends[-1])
    assert lo == 173 and hi == lo + 179 + many
    want = run(q[lo:hi], k[lo:hi], v[lo:hi], ends - lo, dout[lo:hi])
    q, k, v, dout = (t.clone() for t in (q, k, v, dout))
    for t in (q, k, v, dout):
        t[:lo] = t[hi:] = float("nan")
    for x, y in zip(run(q, k, v, ends, dout), want):
        assert torch.equal(x[lo:hi], y) and (x[:lo] == 0).all() and (x[hi:] == 0).all()


@DTYPES
@pytest.mark.parametrize("d", [40, 128, 256])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_scores_of_minus_infinity(causal, d, dtype):
    """Keys whose score is -inf, more of them than any tile holds: no part of the sums.  Rows that
    see no other key are NaN, as a softmax over nothing is."""
    q, k, v, offsets, dout = make([300, 500], 1, 1, d, d, dtype)
    q, k = q.abs() + 1, k.clone()
    k[:280, 0, 0] = -math.inf
    out = run(q, k, v, offsets, dout, causal=causal)[0]
    q0, k0 = q.clone(), k.clone()
    k0[:280, 0, 0] = 0
    S = d ** -0.5 * (q0[:300, 0].double() @ k0[:300, 0].double().T)
    S[:, :280] = -math.inf
    if causal:
        S = S.masked_fill(~torch.ones(300, 300, dtype=torch.bool, device="cuda").tril(), -math.inf)
    want = torch.softmax(S, -1) @ v[:300, 0].double()
    first = 280 if causal else 0
    assert torch.isnan(out[:first]).all() and torch.isfinite(out[first:]).all()
    b = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    err = ((d + 2) * U * d ** -0.5 * (q0[:300, 0].double() @ k0[:300, 0].double().abs().T)).amax()
    r = 2 * err + (8 + 300 + 2 * S[S.isfinite()].abs().amax()) * U
    P, V = torch.softmax(S, -1), v[:300, 0].double()
    lim = (r + b + 300 * U) * (P @ V.abs()) + (b + 4 * U) * want.abs()
    assert ((out[first:300, 0].double() - want[first:]).abs() <= lim[first:]).all()
    assert torch.equal(out[300:], run(q[300:], k[300:], v[300:], offsets[1:] - 300, dout[300:], causal=causal)[0])


@DTYPES
def test_neighbours_do_not_leak(dtype):
    """Infinities and NaN stay in their sequence and key head."""
    q, k, v, offsets, dout = make([70, 100, 45], 4, 2, 50, 50, dtype)
    want = run(q, k, v, offsets, dout)
    k, v = k.clone(), v.clone()
    k[130, 1] = float("nan")  # row 60 of the second sequence
    v[131, 1] = float("inf")
    got = run(q, k, v, offsets, dout)
    for x, y in zip(got, want):
        own = x.shape[1] // 2
        assert torch.equal(x[:70], y[:70]) and torch.equal(x[170:], y[170:])
        assert torch.equal(x[:, :own], y[:, :own])
    assert torch.isnan(got[0][130:170, 2:]).all()


@DTYPES
def test_large_scores(dtype):
    """Scores in the hundreds: a softmax without its running maximum would overflow."""
    q, k, v, offsets, dout = make([200, 64], 2, 2, 64, 64, dtype, spread=60.0)
    check(q, k, v, offsets, dout)


@DTYPES
def test_scale(dtype):
    check(*make([90, 40], 2, 1, 48, 48, dtype), scale=0.03)


@DTYPES
def test_strides_and_offset_types(dtype):
    q, k, v, offsets, dout = make([77, 130], 4, 2, 40, 40, dtype)
    want = run(q, k, v, offsets, dout)
    heads_first = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (q, k, v, dout)]
    odd = [torch.cat([torch.zeros_like(t[..., :1]), t], -1)[..., 1:] for t in (q, k, v)]
    column = [t.permute(0, 2, 1).contiguous().permute(0, 2, 1) for t in (q, k, v)]
    for args in ((*heads_first[:3], offsets, heads_first[3]), (*odd, offsets.to(torch.int32), dout),
                 (*column, offsets, dout)):
        for x, y in zip(run(*args), want):
            assert torch.equal(x, y)


def test_broadcast_keys_get_summed_gradients():
    """One row of keys and values expanded over all rows: autograd sums the rows' gradients."""
    from mygenerativerecommenders_amd import ops
    q, k, v, offsets, dout = make([50, 20], 2, 1, 32, 32, torch.float32)
    k1, v1 = (t[:1].detach().clone().requires_grad_(True) for t in (k, v))
    out = ops.jagged_attention(q, k1.expand_as(k), v1.expand_as(v), offsets)
    gk, gv = torch.autograd.grad(out, (k1, v1), dout)
    _, _, dk, dv = run(q, k1.detach().expand_as(k).contiguous(), v1.detach().expand_as(v).contiguous(), offsets, dout)
    assert torch.allclose(gk, dk.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)
    assert torch.allclose(gv, dv.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


def test_gradients_against_differences():
    """Central differences (h = 1e-2) of the sum along random unit directions.  Their own error:
    h^2 / 6 = 1.7e-5 times a third derivative (of the order of the gradient's norm: scores are
    of order one), and the forward's fp32 error over 2h, about 1e-6 sqrt(outputs) / 2e-2 = 3e-3
    of an output's size at most; the gradients' norms are some tens."""
    from mygenerativerecommenders_amd import ops
    q, k, v, offsets, dout = make([19, 40], 2, 1, 24, 24, torch.float32)
    _, *grads = run(q, k, v, offsets, dout)
    h, gen = 1e-2, torch.Generator(device="cuda").manual_seed(5)
    for i, g in enumerate(grads):
        way = torch.randn(g.shape, device="cuda", generator=gen)
        way /= way.norm()
        side = []
        for sign in (1, -1):
            args = [q, k, v]
            args[i] = args[i] + sign * h * way
            side.append((ops.jagged_attention(*args, offsets).double() * dout.double()).sum())
        diff = ((side[0] - side[1]) / (2 * h)).item()
        assert abs(diff - (g * way).sum().item()) <= 2e-3 * max(1.0, g.norm().item()), i


@DTYPES
def test_same_bits_every_run_and_on_another_stream(dtype):
    args = make([300, 211, 128], 4, 2, 64, 64, dtype)
    want = run(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(*args)
    torch.cuda.current_stream().wait_stream(side)
    for x, y, z in zip(want, got, run(*args)):
        assert torch.equal(x, y) and torch.equal(x, z)


@DTYPES
def test_captured_and_replayed(dtype):
    """Two graphs of forward and backward, replayed in turn with eager work between: each
    replay reads its own inputs' present values."""
    q, k, v, offsets, dout = make([100, 0, 211], 2, 1, 50, 50, dtype, spare=9)
    pairs = []
    for i in range(2):
        bufs = [t.clone() for t in (q, k, v, dout)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*bufs[:3], offsets, bufs[3])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(*bufs[:3], offsets, bufs[3])
        pairs.append((graph, bufs, outs))
    for step in range(4):
        graph, bufs, outs = pairs[step % 2]
        for b, t in zip(bufs, (q, k, v, dout)):
            b.copy_(t * (1 + 0.25 * step))
        graph.replay()
        want = run(*[b.clone() for b in bufs[:3]], offsets, bufs[3].clone())
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y), step


def test_rows_beyond_32_bits():
    """Rows whose element offsets pass 2^31 in their buffer: 60,000 rows 40,000 apart, cut into
    short sequences; the last ones against the formula.  (Bits are not compared with a small
    call's: the number of wave sets that share the sums goes by the number of tiles.)"""
    stride, rows = 40000, 60000
    q, k, v, offsets, dout = make([64, 200], 1, 1, 32, 32, torch.bfloat16)
    ref, lim = reference(q, k, v, offsets, True, 32 ** -0.5, dout)
    big = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda").view(rows, stride)
    views = []
    for i, t in enumerate((q, k, v)):
        view = big[:, 64 * i:64 * i + 32].unflatten(1, (1, 32))
        view[:rows - 264] = 0
        view[rows - 264:] = t
        views.append(view)
    assert views[0].stride(0) == stride
    cut = torch.arange(0, rows - 264, 128, device="cuda")
    ends = torch.cat([cut, torch.tensor([rows - 264, rows - 200, rows], device="cuda")])
    g = torch.zeros(rows, 1, 32, dtype=torch.bfloat16, device="cuda")
    g[rows - 264:] = dout
    for x, y, e in zip(run(*views, ends, g), ref, lim):
        assert ((x[rows - 264:].double() - y).abs() <= e).all()


def test_refusals():
    from mygenerativerecommenders_amd import _lib, ops
    q, k, v, offsets, _ = make([10, 5], 4, 2, 16, 16, torch.float32)
    with pytest.raises(_lib.GrError, match="CPU tensor"):
        ops.jagged_attention(q.cpu(), k, v, offsets)
    with pytest.raises(TypeError):
        ops.jagged_attention(q.half(), k.half(), v.half(), offsets)
    with pytest.raises(TypeError):
        ops.jagged_attention(q, k.bfloat16(), v, offsets)
    for bad in ((q[0], k, v), (q, k[:3], v), (q, k, v[:, :1]), (q[..., :8], k, v), (q[:, :3], k, v), (q[:, :0], k, v)):
        with pytest.raises(ValueError):
            ops.jagged_attention(*bad, offsets)
    wide = torch.zeros(15, 2, 257, device="cuda")
    with pytest.raises(ValueError, match="widths"):
        ops.jagged_attention(wide, wide, wide, offsets)
    for bad in (offsets.float(), offsets[None], offsets[:0]):
        with pytest.raises(ValueError, match="offsets"):
            ops.jagged_attention(q, k, v, bad)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            ops.jagged_attention(q, k, v, offsets, scale=bad)
    q.requires_grad_(True)
    (g,) = torch.autograd.grad(ops.jagged_attention(q, k, v, offsets).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_empty_batches():
    from mygenerativerecommenders_amd import ops
    none = torch.zeros(0, 2, 16, device="cuda", requires_grad=True)
    out = ops.jagged_attention(none, none, none, torch.zeros(3, dtype=torch.int64, device="cuda"))
    out.sum().backward()
    assert out.shape == (0, 2, 16) and none.grad.shape == (0, 2, 16)
    some = torch.randn(9, 2, 16, device="cuda")
    for offsets in (torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")):
        assert (ops.jagged_attention(some, some, some, offsets) == 0).all()


@DTYPES
@pytest.mark.parametrize("d", [40, 128, 256])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_one_row_of_a_wave_overflows_to_minus_infinity(causal, d, dtype):
    """Scores of a few rows overflow to -inf over the first tiles, their neighbours' are ordinary: the
    rows' sums are those of the keys behind, where all their scores are zero."""
    n, first = 300, 140
    _, _, v, offsets, dout = make([n], 1, 1, d, d, dtype)
    q, k = torch.full((n, 1, d), 1e-25, device="cuda").to(dtype), torch.zeros(n, 1, d, device="cuda").to(dtype)
    k[:first] = -1e25
    q[first + 3::37] = 1e30
    S = d ** -0.5 * (q[:, 0].double() @ k[:, 0].double().T)
    S[S < -1e30] = -math.inf
    if causal:
        S = S.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -math.inf)
    err = 2 * (d + 2) * U * d ** 0.5 + (8 + n + 2 * d ** 0.5) * U  # |q k| sums to d
    P, V, b = torch.softmax(S, -1), v[:, 0].double(), 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    lim = (err + b + n * U) * (P @ V.abs()) + (b + 4 * U) * (P @ V).abs() + 1e-30
    out, *grads = run(q, k, v, offsets, dout, causal=causal)
    assert ((out[:, 0].double() - P @ V).abs() <= lim).all()
    assert all(torch.isfinite(t).all() for t in grads)


@DTYPES
@pytest.mark.parametrize("d", [1, 40, 128, 256])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_keys_masked_by_the_lowest_value(causal, d, dtype):
    """A column of ones in q against the type's lowest value in some keys' rows, tiles of them in the
    front: no part of the sums of rows that see another key, forward and backward.  Rows that see no other
    are the mean of what they see, and give no gradient."""
    n = 330
    q, k, v, offsets, dout = make([n], 1, 1, d, d, dtype)
    q, k, dout = q.clone(), k.clone(), dout.clone()
    masked = torch.zeros(n, dtype=torch.bool, device="cuda")
    masked[:150] = masked[200:203] = masked[250:] = True
    q[:, 0, -1] = 1
    k[:, 0, -1] = torch.where(masked, torch.finfo(dtype).min, 0)
    got = run(q, k, v, offsets, dout, causal=causal)
    live = ~masked if not causal else ~masked & torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    some = live.expand(n, n).any(1)
    # the same rows with the masked keys' values out of the way: their probabilities are zero
    k0 = k.clone()
    k0[masked, 0, -1] = 0
    b, s = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0, d ** -0.5
    Q, K, V, G = (t[:, 0].double() for t in (q, k0, v, dout))
    G = G * some[:, None]
    S = s * (Q @ K.T)
    err = (d + 2) * U * s * (Q.abs() @ K.abs().T)
    S = S.masked_fill(~live, -math.inf)
    seen = torch.ones(n, n, dtype=torch.float64, device="cuda")
    seen = (seen.tril() if causal else seen) / (torch.arange(1, n + 1, device="cuda")[:, None] if causal else n)
    P = torch.where(some[:, None], torch.softmax(S, -1), seen)
    r = err + err.amax(1, keepdim=True) + (8 + n + 2 * S.masked_fill(~live, 0).abs().amax(1, keepdim=True)) * U
    O, dP = P @ V, G @ V.T
    eO = (P * (r + b + n * U)) @ V.abs()
    D = (G * O).sum(1, keepdim=True)
    eD = ((b + d * U) * (G * O).abs() + G.abs() * eO).sum(1, keepdim=True)
    dS = P * (dP - D)
    eS = r * dS.abs() + P * (eD + d * U * (G.abs() @ V.abs().T)) + (b + n * U) * dS.abs()
    ref = [(O, eO), (s * (dS @ K), s * (eS @ K.abs())), (s * (dS.T @ Q), s * (eS.T @ Q.abs())),
           (P.T @ G, (P * (r + b + n * U)).T @ G.abs())]
    for name, x, (y, e) in zip(("out", "dq", "dk", "dv"), got, ref):
        assert ((x[:, 0].double() - y).abs() <= e + (b + 4 * U) * y.abs() + 1e-30).all(), name


@DTYPES
def test_contiguous_views_that_start_anywhere(dtype):
    """What torch counts as contiguous and the kernels' 4-byte loads do not take: an odd first element,
    one head with a stride of its own, a single row far from the next."""
    from mygenerativerecommenders_amd import ops
    q, k, v, offsets, dout = make([77, 30], 4, 2, 40, 40, dtype)
    want = run(q, k, v, offsets, dout)

    def odd(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        got = room[1:].view(t.shape)
        return got.copy_(t)

    for i in range(3):
        args = [q, k, v]
        args[i] = odd(args[i])
        assert args[i].is_contiguous() and args[i].data_ptr() % 4 == (2 if dtype == torch.bfloat16 else 0)
        for x, y in zip(run(*args, offsets, dout), want):
            assert torch.equal(x, y)
    for x, y in zip(run(q, k, v, offsets, odd(dout)), want):
        assert torch.equal(x, y)
    # a gradient that autograd cuts out of a longer one
    q1, k1, v1 = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = ops.jagged_attention(q1, k1, v1, offsets)
    joined = torch.cat([torch.zeros(3, dtype=dtype, device="cuda"), out.flatten()])
    for x, y in zip(torch.autograd.grad(joined, (q1, k1, v1), torch.cat([torch.ones_like(joined[:3]), dout.flatten()])), want[1:]):
        assert torch.equal(x, y)
    # one head: its stride is 1
    args = make([50, 13], 1, 1, 40, 40, dtype)
    heads = [t.reshape(63, 40, 1).permute(0, 2, 1) for t in args[:3]]
    assert heads[0].stride(1) == 1
    for x, y in zip(run(*heads, *args[3:]), run(*args)):
        assert torch.equal(x, y)
    # a row of rows 2^22 apart
    one = [t.as_strided(t[:1].shape, ((1 << 22) + 1, *t.stride()[1:])) for t in (q, k, v)]
    ends = torch.tensor([0, 1], device="cuda")
    for x, y in zip(run(*one, ends, dout[:1]), run(*(t[:1].clone() for t in (q, k, v)), ends, dout[:1])):
        assert torch.equal(x, y)


@DTYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("which", ["q", "k", "v", "all"])
@pytest.mark.parametrize("step", [0, 24], ids=["one row for all", "overlapping"])
def test_rows_narrower_than_their_width(step, which, causal, dtype):
    """Rows that are one row, or that share columns with the next: the tile behind a sequence's end
    holds real values then, with scores in the hundreds, and no part of the sums."""
    q, k, v, offsets, dout = make([1, 33, 0, 70, 127], 2, 2, 40, 40, dtype)
    rows = int(offsets[-1])

    def narrow(t):
        flat = (20.0 * t).to(dtype).reshape(-1)
        return flat.as_strided((rows, 2, 40), (step, 40, 1))

    q, k, v = (narrow(t) if which in (n, "all") else t for n, t in zip("qkv", (q, k, v)))
    if which == "q":
        k = (20.0 * k).to(dtype)
    check(q, k, v, offsets, dout, causal=causal)


def test_a_second_derivative_raises_where_it_is_taken():
    """create_graph=True: the first gradient is the same and carries a history that raises, so that no
    term of a sum is left out in silence."""
    from mygenerativerecommenders_amd import ops
    q, k, v, offsets, dout = make([40, 21], 4, 2, 16, 16, torch.float32)
    want = run(q, k, v, offsets, dout)[1:]
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    grads = torch.autograd.grad(ops.jagged_attention(q, k, v, offsets), (q, k, v), dout, create_graph=True)
    for g, w in zip(grads, want):
        assert torch.equal(g, w) and g.requires_grad
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(q.square().sum() + g.square().sum(), q, retain_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        (q.square().sum() + grads[2].square().sum()).backward(retain_graph=True)
    w = dout.clone().requires_grad_(True)  # the product with a gradient's gradient: by way of dout
    (g,) = torch.autograd.grad(ops.jagged_attention(q, k, v, offsets), q, w, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum() + w.sum(), w)
    (gq,) = torch.autograd.grad(q.square().sum() + 0 * grads[0].detach().sum(), q)
    assert torch.equal(gq, 2 * q)


def test_no_derivative_is_dropped_in_silence():
    """Forward-mode derivatives and traces, which the kernels know nothing of, raise; a batched map runs
    them in a loop, a compiled function around them."""
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx
    from mygenerativerecommenders_amd import ops
    q, k, v, offsets, _ = make([10, 5], 4, 2, 16, 16, torch.float32)
    for grad in (False, True):
        with fw.dual_level():
            for i in range(3):
                args = [q, k, v]
                args[i] = fw.make_dual(args[i].clone().requires_grad_(grad), torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    ops.jagged_attention(*args, offsets)
    f = lambda x: ops.jagged_attention(x, k, v, offsets)  # noqa: E731
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(f)(q)
    with pytest.raises(NotImplementedError, match="plain tensors"):
        torch.func.grad(lambda x: f(x).sum())(q)
    assert torch.equal(torch.func.vmap(f)(torch.stack([q, 2 * q])), torch.stack([f(q), f(2 * q)]))
    assert torch.equal(torch.compile(f, backend="eager")(q), f(q))


def test_refuses_offsets_that_32_bits_do_not_count():
    """2^32 + 2 offsets (one element, expanded) are not two."""
    from mygenerativerecommenders_amd import ops
    q, k, v, offsets, _ = make([10, 5], 4, 2, 16, 16, torch.float32)
    for n in (1 << 31, (1 << 32) + 2):
        with pytest.raises(ValueError, match="offsets"):
            ops.jagged_attention(q, k, v, offsets[:1].expand(n))
