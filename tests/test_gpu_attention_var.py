"""Attention with a relative position bias and / or key counts, and the per-head normalisation + rotation pass, against plain
64-bit arithmetic on the same inputs.

Tolerances are bounds, element by element, of the roundings the kernels make (u = half a step of the tensor's type, 2^-8 for
bf16 and 2^-24 for fp32; U = 2^-24 for the arithmetic):
  * a score is a sum of Dh products and a bias, and the exponential's argument is that times log2 e less the row's maximum:
    its error is at most e = (Dh + 8) U (scale |q| |k| + |bias| + |row maximum| + 1), the relative error of a probability 2 e
    (its numerator and the row sum, which has Lk more roundings) plus, for bf16, u for the rounding of the numerators that
    multiply V and u for that of the row sum's terms;
  * o: (that) * (P |V|) + u |o|;       P in the backward, from the stored log-sum-exp: the same relative error r
  * dV: r (P^T |dO|) + u P^T |dO| + u |dV|;   dS = P (dP - delta): r |dS| + P (E + Dh U |dO| |V|), where the error E of
    delta = sum dO o is sum |dO| (error of o as stored);  dS is rounded (u |dS|) before it multiplies K or Q;
  * the bias gradient sums dS itself over samples and pairs in 32 bits: n U sum |dS| on top."""
import math

import pytest
import torch

from vit_amd import RelativeBuckets, qk_norm_rope
from vit_amd.attention import attention

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from vit_amd import kernels as K

DEV = "cuda"
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, k, v, scale, bias, lens, dout=None, keep=None, dropped=None):
    """64-bit results and error bounds.  q, k, v [B, L, H, Dh]; bias [H, Lq, Lk] or None; lens: list or None; ``keep``: 0 or
    1 / (1 - p) per probability.  Returns {name: (value, bound)}."""
    u = half_step(q.dtype)
    low = q.dtype == torch.bfloat16
    Q, Kk, V = [t.detach().double().cpu().transpose(1, 2) for t in (q, k, v)]   # [B, H, L, Dh]
    B, H, Lq, Dh = Q.shape
    Lk = Kk.shape[2]
    lens = [Lk] * B if lens is None else [min(max(n, 0), Lk) for n in lens]
    live = (torch.arange(Lk)[None] < torch.tensor(lens)[:, None])[:, None, None]
    Kk, V = Kk.masked_fill(~live.transpose(2, 3), 0.0), V.masked_fill(~live.transpose(2, 3), 0.0)
    bias = torch.zeros(1, 1, 1, dtype=torch.float64) if bias is None else bias.double().cpu()
    s = scale * Q @ Kk.transpose(-1, -2) + bias
    s = s.masked_fill(~live, -math.inf)
    m = s.amax(-1, keepdim=True) if Lk else s.new_full((B, H, Lq, 1), -math.inf)
    m0 = m.masked_fill(m == -math.inf, 0.0)
    e = torch.exp(s - m0)
    l = e.sum(-1, keepdim=True)
    P = e / l.masked_fill(l == 0, 1.0)
    fin = bias.masked_fill(bias == -math.inf, 0.0).abs()
    es = (Dh + 8) * U * (scale * Q.abs() @ Kk.abs().transpose(-1, -2) + fin + m0.abs() + 1.0)
    es = es.clamp_max(1.0) * (P > 0)   # only where there is a probability (a huge bias elsewhere does not matter)
    worst = es.amax(-1, keepdim=True) if Lk else es.new_zeros((B, H, Lq, 1))
    r = 2 * es + 2 * worst + (Lk + 8) * U + (2 * u if low else 0.0)   # relative error of a probability
    kp = torch.ones(()) if keep is None else keep.double().cpu()
    Pd = P * kp
    o = Pd @ V
    eo = (Pd * r) @ V.abs() + u * o.abs()
    back = lambda t: t.transpose(1, 2)
    out = {"o": (back(o), back(eo))}
    if dout is not None:
        G = dout.double().cpu().transpose(1, 2)
        dV = Pd.transpose(-1, -2) @ G
        edV = (Pd * (r + (u if low else 0.0))).transpose(-1, -2) @ G.abs() + u * dV.abs()
        delta = (G * o).sum(-1, keepdim=True)
        E = (G.abs() * eo).sum(-1, keepdim=True) + Dh * U * (G.abs() * o.abs()).sum(-1, keepdim=True)
        dP = G @ V.transpose(-1, -2) * kp
        dS = P * (dP - delta)
        eS = r * dS.abs() + P * (E + (Dh + 4) * U * (G.abs() @ V.abs().transpose(-1, -2) * kp + delta.abs()))
        # second-order term: probabilities off by r multiply a dP - delta off by E; r <= 1/16 covers it
        eS = eS * (1 + 1 / 16)
        eSr = eS + (u if low else 0.0) * dS.abs()
        sums = (Lk + 8) * U
        dQ, dK = scale * dS @ Kk, scale * dS.transpose(-1, -2) @ Q
        out["dq"] = (back(dQ), back(scale * (eSr + sums * dS.abs()) @ Kk.abs() + u * dQ.abs()))
        out["dk"] = (back(dK), back(scale * (eSr + (Lq + 8) * U * dS.abs()).transpose(-1, -2) @ Q.abs() + u * dK.abs()))
        out["dv"] = (back(dV), back(edV + (Lq + 8) * U * Pd.transpose(-1, -2) @ G.abs()))
        out["dS"] = (dS, eS)
    return out


def bucket_sums(dS, eS, index, nb, dtype):
    """Gradient of the bias table [nb, H] and its bound from dS [B, H, Lq, Lk]."""
    H = dS.shape[1]
    flat = index.reshape(-1).cpu().long()

    def sums(t):
        return torch.zeros(nb, H, dtype=torch.float64).index_add_(0, flat, t.sum(0).reshape(H, -1).t().contiguous())

    n = dS.shape[0] * flat.numel()
    val = sums(dS)
    return val, sums(eS) + min(n, 4096) * U * sums(dS.abs()) + half_step(dtype) * val.abs()


def check(got, want, name):
    val, bound = want
    got = got.detach().double().cpu()
    assert got.shape == val.shape, (name, got.shape, val.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    err = (got - val).abs()
    over = err - bound
    at = int(over.argmax()) if over.numel() else 0
    assert bool((over <= 1e-30).all()), f"{name}: error {err.reshape(-1)[at]:.3e} beyond its bound {bound.reshape(-1)[at]:.3e} at {at}"


def make(B, Lq, Lk, H, Dh, dtype, seed, packed):
    """q, k, v: views of packed projections (or tensors of their own), and the output's gradient."""
    g = torch.Generator().manual_seed(seed)
    if packed:
        q = torch.randn(B, Lq, H, Dh, generator=g).to(DEV, dtype)
        kv = torch.randn(B, Lk, 2, H, Dh, generator=g).to(DEV, dtype)
        k, v = kv[:, :, 0], kv[:, :, 1]
    else:   # heads outside the rows, every tensor with strides of its own
        q = torch.randn(B, H, Lq, Dh, generator=g).to(DEV, dtype).transpose(1, 2)
        k = torch.randn(H, B, Lk, Dh, generator=g).to(DEV, dtype).permute(1, 2, 0, 3)
        v = torch.randn(B, Lk, H, Dh, generator=g).to(DEV, dtype)
    return q, k, v, torch.randn(B, Lq, H, Dh, generator=g).to(DEV, dtype)


def run(q, k, v, dout, algo, **kw):
    old = K.set_algo(algo)
    try:
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        table = kw.pop("bias_table", None)
        if table is not None:
            table = table.detach().requires_grad_(True)
            leaves.append(table)
        o = attention(*leaves[:3], bias_table=table, **kw)
        grads = torch.autograd.grad(o, leaves, dout)
        with torch.no_grad():
            again = attention(q, k, v, bias_table=table, **kw)
        assert torch.equal(o, again), "the call without gradients gives other values"
    finally:
        K.set_algo(old)
    return dict(zip(("o", "dq", "dk", "dv", "dtable"), (o, *grads)))


SHAPES = [   # B, Lq, Lk, H, Dh: one row, one key, tile borders and their neighbours, few and many rows
    (1, 1, 1, 1, 64), (2, 1, 65, 3, 64), (2, 3, 300, 2, 32), (1, 32, 64, 2, 64), (2, 33, 63, 1, 88), (1, 64, 129, 2, 80),
    (1, 65, 31, 3, 96), (2, 127, 128, 1, 128), (1, 197, 197, 2, 64), (2, 272, 272, 1, 64), (1, 130, 577, 1, 40), (1, 5, 1100, 2, 72),
    (3, 31, 5, 2, 8),
]


@pytest.mark.parametrize("algo", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_relative_bias(shape, dtype, algo):
    B, Lq, Lk, H, Dh = shape
    q, k, v, dout = make(B, Lq, Lk, H, Dh, dtype, Lq * 7 + Lk, packed=Lq % 2 == 1)
    g = torch.Generator().manual_seed(Lk)
    nb = max(1, min(50, Lq * Lk // 2))
    index = torch.randint(0, nb, (Lq, Lk), generator=g)
    table = torch.randn(nb, H, generator=g).to(DEV, dtype)
    got = run(q, k, v, dout, algo, bias_table=table, buckets=RelativeBuckets(index, nb).to(DEV))
    bias = table.double().cpu()[index].permute(2, 0, 1)
    want = reference(q, k, v, Dh ** -0.5, bias, None, dout)
    want["dtable"] = bucket_sums(*want.pop("dS"), index, nb, dtype)
    for n, w in want.items():
        check(got[n], w, n)


@pytest.mark.parametrize("algo", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_key_counts_and_poisoned_padding(shape, dtype, algo):
    """Counts of 0, 1, tile borders, all and (clamped) more and fewer; the padding holds NaN and infinities, which neither
    the outputs nor any gradient may see; the gradients of padding are zeros."""
    _, Lq, Lk, H, Dh = shape
    lens = sorted({0, 1, min(32, Lk), min(33, Lk), max(Lk - 1, 0), Lk}) + [Lk + 5, -3]
    B = len(lens)
    q, k, v, dout = make(B, Lq, Lk, H, Dh, dtype, Lq + Lk * 3, packed=Lq % 2 == 0)
    want = reference(q, k, v, 0.3, None, lens, dout)
    want.pop("dS")
    for b, n in enumerate(lens):
        k[b, max(n, 0):], v[b, max(n, 0):] = float("nan"), float("inf")
    got = run(q, k, v, dout, algo, kv_lengths=torch.tensor(lens, device=DEV, dtype=torch.int64 if Lq % 2 else torch.int32), scale=0.3)
    for n, w in want.items():
        check(got[n], w, n)
    for b, n in enumerate(lens):
        assert not got["dk"][b, max(n, 0):].any() and not got["dv"][b, max(n, 0):].any()
        if n <= 0:
            assert not got["o"][b].any() and not got["dq"][b].any()


@pytest.mark.parametrize("algo", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("L,few", [(70, False), (200, False), (700, True)])
def test_bias_that_masks(dtype, algo, L, few):
    """Buckets of -inf, of the type's lowest value and of its largest: rows left with nothing, rows of nothing but lowest
    values (uniform over them), rows with one key; together with key counts."""
    H, Dh = 2, 64
    Lq = 4 if few else L
    q, k, v, dout = make(2, Lq, L, H, Dh, dtype, L, packed=True)
    lowest = torch.finfo(dtype).min
    table = torch.tensor([[0.5, -0.25], [-math.inf, -math.inf], [lowest, lowest], [30.0, -30.0]]).to(DEV, dtype)
    index = torch.randint(0, 4, (Lq, L), generator=torch.Generator().manual_seed(1))
    index[0] = 1              # nothing left
    index[1] = 2              # all at the lowest value
    index[2] = 1
    index[2, L // 2] = 0      # one key
    index[3, : L // 2] = 1    # the first half masked
    lens = [L, L - 3]
    got = run(q, k, v, dout, algo, bias_table=table, buckets=RelativeBuckets(index, 4).to(DEV),
              kv_lengths=torch.tensor(lens, device=DEV, dtype=torch.int32))
    bias = table.double().cpu().clamp(min=-1e37)[index].permute(2, 0, 1)   # what the kernels make of the lowest value
    bias = torch.where(table.double().cpu()[index].permute(2, 0, 1) == -math.inf, -math.inf, bias)
    # a row at the lowest value only: the scores vanish beside it in 32 bits, the probabilities are equal
    sc = bias.clone()
    want = reference(q, k, v, Dh ** -0.5, sc, lens, dout)
    val, bound = want["o"]
    uniform = torch.stack([v[b, :n].double().mean(0) for b, n in enumerate(lens)]).cpu()
    assert not got["o"][:, 0].any() and not got["dq"][:, 0].any()
    u = half_step(dtype)
    err = (got["o"][:, 1].double().cpu() - uniform).abs()
    assert bool((err <= (3 * u + 2 * L * U) * torch.stack([v[b, :n].double().abs().mean(0) for b, n in enumerate(lens)]).cpu() + 1e-30).all())
    rows = [i for i in range(Lq) if i != 1]
    check(got["o"][:, rows], (val[:, rows], bound[:, rows]), "o")
    check(got["dq"][:, rows], tuple(t[:, rows] for t in want["dq"]), "dq")
    for n in ("dk", "dv", "dtable"):
        assert torch.isfinite(got[n]).all(), n


@pytest.mark.parametrize("algo", [0, 1])
@pytest.mark.parametrize("few", [False, True])
def test_dropout_masks_agree_with_the_gradients(algo, few):
    """V = unit vectors shows the dropped probabilities; the gradients are those of that very mask, and the share of kept
    probabilities is 1 - p."""
    B, H, L, p = 2, 2, 64, 0.3
    Lq = 3 if few else 90
    q, k, _, dout = make(B, Lq, L, H, 64, torch.bfloat16, 5, packed=True)
    v = torch.eye(64, device=DEV, dtype=torch.bfloat16)[None, :, None].expand(B, 64, H, 64).contiguous()
    index = torch.randint(0, 9, (Lq, L), generator=torch.Generator().manual_seed(2))
    plan = RelativeBuckets(index, 9).to(DEV)
    table = torch.randn(9, H, device=DEV, dtype=torch.bfloat16)
    gen = torch.cuda.default_generators[torch.cuda.current_device()]

    def once(algo):
        torch.cuda.manual_seed(11)
        old = K.set_algo(algo)
        try:
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
            o = attention(*leaves[:3], bias_table=leaves[3], buckets=plan, dropout=p, training=True)
            return o, torch.autograd.grad(o, leaves, dout)
        finally:
            K.set_algo(old)

    o, grads = once(algo)
    shown = o.detach().double().cpu().transpose(1, 2)
    keep = (shown > 0).double() / (1 - p)
    share = (shown > 0).double().mean().item()
    n = shown.numel()
    assert abs(share - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n) + 1e-3
    want = reference(q, k, v, 64 ** -0.5, table.double().cpu()[index].permute(2, 0, 1), None, dout, keep=keep)
    dS = want.pop("dS")
    want["dtable"] = bucket_sums(*dS, index, 9, torch.bfloat16)
    for name, t in zip(("o", "dq", "dk", "dv", "dtable"), (o, *grads)):
        check(t, want[name], name)
    other, _ = once(1 - algo)
    assert torch.equal(other > 0, o > 0)   # both kernel families draw the same mask
    assert gen.get_offset() >= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_results_repeat_bit_for_bit(dtype):
    B, Lq, Lk, H, Dh = 3, 150, 333, 4, 64
    q, k, v, dout = make(B, Lq, Lk, H, Dh, dtype, 9, packed=True)
    index = torch.randint(0, 33, (Lq, Lk), generator=torch.Generator().manual_seed(3))
    kw = dict(bias_table=torch.randn(33, H, device=DEV, dtype=dtype), buckets=RelativeBuckets(index, 33).to(DEV),
              kv_lengths=torch.tensor([333, 0, 70], device=DEV))
    first = run(q, k, v, dout, 0, **kw)
    for _ in range(3):
        again = run(q, k, v, dout, 0, **kw)
        for n in first:
            assert torch.equal(first[n], again[n]), n


def test_gradients_against_differences():
    """Central differences of a fixed linear functional of o in fp32: dq, dk, dv and the table's gradient along random
    directions.  Step h = 2^-7 in every direction of unit components: the functional's third derivative is bounded by its
    own size times (direction scores)^3, which the 5e-3 relative term covers; fp32 noise is 2^-20 * |f| / h."""
    B, Lq, Lk, H, Dh = 2, 9, 40, 2, 16
    q, k, v, dout = make(B, Lq, Lk, H, Dh, torch.float32, 21, packed=True)
    index = torch.randint(0, 5, (Lq, Lk), generator=torch.Generator().manual_seed(4))
    plan, table = RelativeBuckets(index, 5).to(DEV), torch.randn(5, H, device=DEV)
    lens = torch.tensor([40, 17], device=DEV)
    got = run(q, k, v, dout, 0, bias_table=table, buckets=plan, kv_lengths=lens)
    ins = dict(q=q, k=k, v=v, table=table)
    h = 2.0 ** -7

    def f(**ch):
        t = {**ins, **ch}
        o = attention(t["q"], t["k"], t["v"], bias_table=t["table"], buckets=plan, kv_lengths=lens)
        return (o.double() * dout.double()).sum().item()

    for n, x in ins.items():
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(6)).to(DEV) / 4
        num = (f(**{n: x + h * d}) - f(**{n: x - h * d})) / (2 * h)
        ana = (got["d" + n].double() * d.double()).sum().item()
        size = (got["d" + n].double() * d.double()).abs().sum().item()
        assert abs(num - ana) <= 5e-3 * size, (n, num, ana)


def test_graph_replays_follow_new_inputs_and_two_graphs_live_side_by_side():
    """Forward and backward captured twice, with other sizes; eager work of other sizes between replays; every replay equals
    the eager result on the inputs copied in before it."""
    def case(Lq, Lk, seed):
        q, k, v, dout = make(2, Lq, Lk, 2, 64, torch.bfloat16, seed, packed=True)
        index = torch.randint(0, 20, (Lq, Lk), generator=torch.Generator().manual_seed(seed))
        return dict(q=q, k=k, v=v, dout=dout, table=torch.randn(20, 2, device=DEV, dtype=torch.bfloat16),
                    plan=RelativeBuckets(index, 20).to(DEV), lens=torch.tensor([Lk, Lk // 2], device=DEV, dtype=torch.int32))

    def step(c):
        leaves = [c[n].detach().requires_grad_(True) for n in ("q", "k", "v", "table")]
        o = attention(*leaves[:3], bias_table=leaves[3], buckets=c["plan"], kv_lengths=c["lens"])
        return [o.detach(), *torch.autograd.grad(o, leaves, c["dout"])]

    cases = [case(4, 500, 1), case(140, 200, 2)]
    graphs = []
    for c in cases:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(c)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(c)
        graphs.append((g, out))
    for rep in range(4):
        wants = []
        for c in cases:
            for n in ("q", "k", "v", "dout", "table"):
                c[n].copy_(torch.randn_like(c[n]))
            c["lens"].copy_(torch.tensor([rep, c["k"].shape[1] - rep], device=DEV))
            wants.append([t.clone() for t in step(c)])
        step(case(33, 77, rep))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (g, out), want in zip(graphs, wants):
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_side_stream_and_concurrent_streams():
    q, k, v, dout = make(2, 100, 300, 4, 64, torch.bfloat16, 31, packed=True)
    index = torch.randint(0, 20, (100, 300), generator=torch.Generator().manual_seed(3))
    kw = dict(bias_table=torch.randn(20, 4, device=DEV, dtype=torch.bfloat16), buckets=RelativeBuckets(index, 20).to(DEV))
    want = run(q, k, v, dout, 0, **kw)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(run(q, k, v, dout, 0, **kw))
    torch.cuda.synchronize()
    for got in outs:
        for n in want:
            assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("Lq", [1, 40])
def test_offsets_beyond_32_bits(Lq):
    """A memory whose second sample starts more than 2^31 elements behind the first."""
    H, Dh, Lk = 2, 64, 100
    gap = 2 ** 31 + 4096
    g = torch.Generator().manual_seed(1)
    buf = torch.empty(gap + Lk * 2 * H * Dh, device=DEV, dtype=torch.bfloat16)
    kv = buf.as_strided((2, Lk, 2, H, Dh), (gap, 2 * H * Dh, H * Dh, Dh, 1))
    kv.copy_(torch.randn(2, Lk, 2, H, Dh, generator=g))
    q = torch.randn(2, Lq, H, Dh, generator=g).to(DEV, torch.bfloat16)
    dout = torch.randn(2, Lq, H, Dh, generator=g).to(DEV, torch.bfloat16)
    lens = [100, 37]
    got = run(q, kv[:, :, 0], kv[:, :, 1], dout, 0, kv_lengths=torch.tensor(lens, device=DEV))
    want = reference(q, kv[:, :, 0], kv[:, :, 1], Dh ** -0.5, None, lens, dout)
    want.pop("dS")
    for n, w in want.items():
        check(got[n], w, n)


def test_unaligned_and_odd_heads():
    """Head sizes and offsets the matrix-unit kernels do not take go to the portable ones (or through one copy)."""
    g = torch.Generator().manual_seed(8)
    for Dh, off in ((12, 0), (1, 0), (20, 3), (64, 1)):
        base = [torch.randn(2, 30, 3, Dh + 8, generator=g).to(DEV, torch.bfloat16) for _ in range(3)]
        q, k, v = [t[..., off:off + Dh] for t in base]
        dout = torch.randn(2, 30, 3, Dh, generator=g).to(DEV, torch.bfloat16)
        got = run(q, k, v, dout, 0, kv_lengths=torch.tensor([30, 11], device=DEV))
        want = reference(q, k, v, Dh ** -0.5, None, [30, 11], dout)
        want.pop("dS")
        for n, w in want.items():
            check(got[n], w, n)


def test_empty_calls():
    for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k = torch.randn(B, Lq, 2, 16, device=DEV), torch.randn(B, Lk, 2, 16, device=DEV)
        leaves = [t.requires_grad_(True) for t in (q, k, k.detach().clone())]
        o = attention(*leaves)
        assert o.shape == q.shape and not o.any()
        for t, g in zip(leaves, torch.autograd.grad(o, leaves, torch.ones_like(o))):
            assert g.shape == t.shape and not g.any()


def test_table_in_another_dtype_keeps_its_own_gradient():
    q, k, v, dout = make(1, 20, 20, 2, 32, torch.bfloat16, 3, packed=True)
    index = torch.arange(400).view(20, 20) % 7
    plan = RelativeBuckets(index, 7).to(DEV)
    table = torch.randn(7, 2, device=DEV)
    low = run(q, k, v, dout, 0, bias_table=table.bfloat16(), buckets=plan)
    own = run(q, k, v, dout, 0, bias_table=table, buckets=plan)
    assert torch.equal(low["o"], own["o"]) and own["dtable"].dtype == torch.float32
    assert torch.equal(own["dtable"].bfloat16(), low["dtable"])


def test_second_derivatives_are_refused():
    q = torch.randn(1, 3, 1, 16, device=DEV, requires_grad=True)
    o = attention(q, q, q)
    (g,) = torch.autograd.grad(o.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- per-head normalisation + rotation --------------------------------------------------------------------------------------
def norm_rope_reference(x, w, b, table, ln, eps, dy):
    """64-bit y, dx, dw, db of one section with their bounds.  x, dy [B, L, H, Dh]; table [2, N, Dh] or [2, B, N, Dh].
    The statistics carry (Dh + 8) U relative errors, the element-wise steps a few U each: 4 (Dh + 16) U of the magnitudes
    covers them; then half a step for the store."""
    u = half_step(x.dtype)
    X = x.detach().double().cpu().requires_grad_(True)
    W = w.detach().double().cpu().requires_grad_(True)
    Bv = None if b is None else b.detach().double().cpu().requires_grad_(True)
    mean = X.mean(-1, keepdim=True) if ln else 0.0
    xc = X - mean
    rstd = (xc.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = xc * rstd * W
    if b is not None:
        n = n + Bv
    Dh, Ln = X.shape[-1], X.shape[1]
    h = Dh // 2
    sin, cos = torch.zeros(X.shape[0], Ln, Dh, dtype=torch.float64), torch.ones(X.shape[0], Ln, Dh, dtype=torch.float64)
    if table is not None:
        N = table.shape[-2]
        sin[:, Ln - N:], cos[:, Ln - N:] = table[0].double().cpu(), table[1].double().cpu()
    sin, cos = sin[:, :, None], cos[:, :, None]
    swap = lambda t: torch.cat([t[..., h:], t[..., :h]], -1)
    y = n * cos + torch.cat([-n[..., h:], n[..., :h]], -1) * sin
    c = 4 * (Dh + 16) * U
    mag = lambda t, sn, cs: t.abs() * cs.abs() + swap(t.abs()) * sn.abs()
    xmag = (X.abs() + (X.abs().mean(-1, keepdim=True) if ln else 0.0)) * rstd   # what cancels in x - mean
    nmag = xmag * W.abs() + (0 if b is None else Bv.abs())
    out = {"y": (y.detach(), (c * mag(nmag, sin, cos) + u * y.abs()).detach())}
    G = dy.double().cpu()
    leaves = [X, W] + ([Bv] if b is not None else [])
    grads = torch.autograd.grad(y, leaves, G)
    dn = (G.abs() * cos.abs() + swap(G.abs() * sin.abs())).detach()
    uu = dn * W.detach().abs()
    xh = xmag.detach()
    rows = X.shape[0] * Ln * X.shape[2]
    # LayerNorm rows with little spread amplify the error of the mean: xh holds that magnitude
    dxm = (rstd * (uu + xh * (uu * xh).mean(-1, keepdim=True) * (1 + xh) + uu.mean(-1, keepdim=True))).detach()
    out["dx"] = (grads[0], 4 * c * dxm * (1 + xh) + u * grads[0].abs())
    cw = c + min(rows, 4096) * U
    out["dw"] = (grads[1], 4 * cw * (dn * xh).sum((0, 1, 2)) + half_step(w.dtype) * grads[1].abs())
    if b is not None:
        out["db"] = (grads[2], 4 * cw * dn.sum((0, 1, 2)) + half_step(w.dtype) * grads[2].abs())
    return out


def rope_table(n, Dh, seed, batch=None):
    g = torch.Generator().manual_seed(seed)
    shape = (n, Dh) if batch is None else (batch, 1, n, Dh)
    ang = torch.rand(shape, generator=g, dtype=torch.float64) * 6.28
    return torch.stack([ang.sin(), ang.cos()]).float().to(DEV)


@pytest.mark.parametrize("ln", [False, True], ids=["rms", "ln"])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("case", [   # B, Lq, Lk, Hq, Hk, Dh, rotated rows of q and k, per-sample tables
    (1, 1, 1, 1, 1, 64, 1, 1, False), (2, 37, 37, 3, 3, 80, 36, 36, False), (1, 50, 7, 5, 2, 88, 50, 0, False),
    (3, 5, 11, 2, 4, 128, 3, 9, True), (2, 130, 64, 1, 9, 96, 130, 60, False), (2, 9, 3, 12, 6, 32, 0, 0, False),
    (1, 20, 20, 2, 2, 8, 20, 20, True), (2, 6, 5, 3, 1, 40, 2, 5, False), (1, 3, 0, 17, 2, 72, 1, 0, False)])
def test_qk_norm_rope(case, dtype, wdtype, ln):
    B, Lq, Lk, Hq, Hk, Dh, nq, nk, per = case
    g = torch.Generator().manual_seed(Lq * 31 + Dh)
    wide = torch.randn(B, Lq, 3, Hq, Dh, generator=g).to(DEV, dtype)
    q, k = wide[:, :, 1], torch.randn(B, Hk, Lk, Dh, generator=g).to(DEV, dtype).transpose(1, 2)
    w = [(1 + 0.3 * torch.randn(Dh, generator=g)).to(DEV, wdtype) for _ in range(2)]
    b = [(0.3 * torch.randn(Dh, generator=g)).to(DEV, wdtype) if ln else None for _ in range(2)]
    tables = [rope_table(n, Dh, 3 + i, B if per else None) if n else None for i, n in enumerate((nq, nk))]
    dq, dk = torch.randn(B, Lq, Hq, Dh, generator=g).to(DEV, dtype), torch.randn(B, Lk, Hk, Dh, generator=g).to(DEV, dtype)
    leaves = {n: t.detach().requires_grad_(True) for n, t in dict(q=q, k=k, wq=w[0], wk=w[1], bq=b[0], bk=b[1]).items() if t is not None}
    args = (leaves["q"], leaves["k"], leaves["wq"], leaves["wk"], leaves.get("bq"), leaves.get("bk"))
    yq, yk = qk_norm_rope(*args, rope_q=tables[0], rope_k=tables[1], eps=1e-4, use_layer_norm=ln)
    grads = dict(zip(leaves, torch.autograd.grad([yq, yk], list(leaves.values()), [dq, dk])))
    with torch.no_grad():
        for a, b_ in zip(qk_norm_rope(*args, rope_q=tables[0], rope_k=tables[1], eps=1e-4, use_layer_norm=ln), (yq, yk)):
            assert torch.equal(a, b_)
        only, none = qk_norm_rope(q, None, w[0], None, b[0], rope_q=tables[0], eps=1e-4, use_layer_norm=ln)
        assert none is None and torch.equal(only, yq)
    for s, x, y, i, dy in (("q", q, yq, 0, dq), ("k", k, yk, 1, dk)):
        t = tables[i]
        want = norm_rope_reference(x, w[i], b[i], t if t is None or t.dim() == 3 else t[:, :, 0], ln, 1e-4, dy)
        check(y, want["y"], s)
        check(grads[s], want["dx"], "d" + s)
        check(grads["w" + s], want["dw"], "dw" + s)
        if ln:
            check(grads["b" + s], want["db"], "db" + s)


def test_qk_norm_rope_in_place_strided_and_wide_batches():
    """In place on the packed projection, heads wider apart than they are long, enough rows for several steps of every wave;
    heads off the 16-byte boundaries are refused by the kernel and copied by the public call."""
    g = torch.Generator().manual_seed(5)
    off = torch.randn(2, 9, 3, 84, generator=g).to(DEV, torch.bfloat16)[..., :80]
    w80 = torch.ones(80, device=DEV)
    with pytest.raises(RuntimeError, match="16 bytes"):
        K.qk_norm_rope_fwd(off, None, torch.empty_like(off), None, (w80, None), (None, None), (None, None), 1e-5, False)
    check(qk_norm_rope(off, None, w80)[0], norm_rope_reference(off, w80, None, None, False, 1e-5, torch.zeros(2, 9, 3, 80))["y"], "copied")
    for Dh, pad, B, Ln in ((80, 8, 3, 50), (64, 0, 40, 300), (24, 0, 5, 700), (16, 8, 2, 40)):
        buf = torch.randn(B, Ln, 2, 3, Dh + pad, generator=g).to(DEV, torch.bfloat16)
        x = buf[..., :Dh]
        w = (1 + 0.3 * torch.randn(Dh, generator=g)).to(DEV)
        t = rope_table(Ln, Dh, 9)
        want = [norm_rope_reference(x[:, :, i], w, None, t, False, 1e-5, torch.zeros(B, Ln, 3, Dh))["y"] for i in range(2)]
        rest = buf[..., Dh:].clone()
        K.qk_norm_rope_fwd(x[:, :, 0], x[:, :, 1], x[:, :, 0], x[:, :, 1], (w, w), (None, None), (t, t), 1e-5, False)
        for i in range(2):
            check(x[:, :, i], want[i], "in place")
        assert torch.equal(buf[..., Dh:], rest)


# ---- variants that only some sizes reach ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H", [1, 2, 4, 6, 8, 12])
@pytest.mark.parametrize("B,Lq,Lk", [(5, 2, 300), (5, 140, 150), (2, 70, 1100), (1, 300, 40)])
def test_head_counts_shares_and_key_ranges(B, Lq, Lk, H, dtype):
    """Head counts that lay the bias out 1, 2, 4 and 8 at a time and group 1, 2 and 4 heads of few queries; samples shared out
    in the bias gradient; key ranges shared out in the forward pass; all with counts."""
    q, k, v, dout = make(B, Lq, Lk, H, 64, dtype, H + Lq, packed=H % 4 == 0)
    index = torch.randint(0, 21, (Lq, Lk), generator=torch.Generator().manual_seed(H))
    table = torch.randn(21, H, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
    lens = [Lk, Lk // 2, 0, Lk - 1, 33][:B]
    got = run(q, k, v, dout, 0, bias_table=table, buckets=RelativeBuckets(index, 21).to(DEV),
              kv_lengths=torch.tensor(lens, device=DEV, dtype=torch.int32))
    want = reference(q, k, v, 64 ** -0.5, table.double().cpu()[index].permute(2, 0, 1), lens, dout)
    want["dtable"] = bucket_sums(*want.pop("dS"), index, 21, dtype)
    for n, w in want.items():
        check(got[n], w, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,Lq,Lk,H,Dh", [(1100, 1, 40, 4, 32), (1100, 1, 40, 2, 64), (4200, 1, 33, 1, 64), (64, 40, 50, 8, 32), (64, 33, 200, 8, 96)])
def test_many_samples(B, Lq, Lk, H, Dh, dtype):
    """Enough samples that no axis is shared out; empty, single-key and full memories among them."""
    q, k, v, dout = make(B, Lq, Lk, H, Dh, dtype, B, packed=True)
    lens = torch.randint(0, Lk + 1, (B,), generator=torch.Generator().manual_seed(1))
    lens[:3] = torch.tensor([0, 1, Lk])
    got = run(q, k, v, dout, 0, kv_lengths=lens.to(DEV))
    want = reference(q, k, v, Dh ** -0.5, None, lens.tolist(), dout)
    want.pop("dS")
    for n, w in want.items():
        check(got[n], w, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Lq", [1, 40, 70])
def test_expanded_operands(Lq, dtype):
    """Queries expanded over rows (a stride of 0) and over samples, keys over heads, the output's gradient over everything:
    rows beyond the last must not be read as more of them; gradients of what was expanded are sums."""
    B, Lk, H, Dh = 3, 90, 4, 64
    g = torch.Generator().manual_seed(Lq)
    q1 = torch.randn(1, 1, H, Dh, generator=g).to(DEV, dtype).requires_grad_(True)
    k1 = torch.randn(B, Lk, 1, Dh, generator=g).to(DEV, dtype).requires_grad_(True)
    v = torch.randn(B, Lk, H, Dh, generator=g).to(DEV, dtype).requires_grad_(True)
    d1 = torch.randn(1, 1, 1, Dh, generator=g).to(DEV, dtype)
    lens = [90, 41, 0]
    o = attention(q1.expand(B, Lq, H, Dh), k1.expand(B, Lk, H, Dh), v, kv_lengths=torch.tensor(lens, device=DEV))
    dout = d1.expand(B, Lq, H, Dh)
    got = torch.autograd.grad(o, (q1, k1, v), dout)
    want = reference(q1.expand(B, Lq, H, Dh), k1.expand(B, Lk, H, Dh), v, Dh ** -0.5, None, lens, dout)
    check(o, want["o"], "o")
    check(got[2], want["dv"], "dv")
    u = half_step(dtype)
    for name, x, dims in (("dq", got[0], (0, 1)), ("dk", got[1], (2,))):
        val, bound = want[name]
        n = math.prod(val.shape[d] for d in dims)
        # the sum over the expanded axes is torch's, in 32 bits, rounded once
        total = (bound + n * U * val.abs()).sum(dims, keepdim=True) + u * val.sum(dims, keepdim=True).abs()
        check(x, (val.sum(dims, keepdim=True), total), name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,Lq,H", [(2, 1, 2), (3, 33, 1), (2, 130, 2), (70, 1, 8)])
def test_dropout_gradients_for_any_row_count(B, Lq, H, dtype):
    """As above, the mask read off V = unit vectors: one query (whose rows have no stride), some, many."""
    p = 0.25
    q, k, _, dout = make(B, Lq, 64, H, 64, dtype, 5 + Lq, packed=Lq % 2 == 0)
    v = torch.eye(64, device=DEV, dtype=dtype)[None, :, None].expand(B, 64, H, 64).contiguous()
    index = torch.randint(0, 9, (Lq, 64), generator=torch.Generator().manual_seed(2))
    table = torch.randn(9, H, device=DEV, dtype=dtype)
    torch.cuda.manual_seed(12)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    o = attention(*leaves[:3], bias_table=leaves[3], buckets=RelativeBuckets(index, 9).to(DEV), dropout=p, training=True)
    grads = torch.autograd.grad(o, leaves, dout)
    keep = (o.detach().double().cpu().transpose(1, 2) > 0).double() / (1 - p)
    want = reference(q, k, v, 64 ** -0.5, table.double().cpu()[index].permute(2, 0, 1), None, dout, keep=keep)
    want["dtable"] = bucket_sums(*want.pop("dS"), index, 9, dtype)
    for name, t in zip(("o", "dq", "dk", "dv", "dtable"), (o, *grads)):
        check(t, want[name], name)


@pytest.mark.parametrize("algo", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Lq", [3, 100])
def test_gradients_of_rows_at_the_lowest_value(Lq, dtype, algo):
    """Beside the type's lowest value the scores vanish in 32 bits: such rows weigh their keys equally, as rows of zero queries
    without a bias do, and their gradients (but dk, which multiplies the queries) are those."""
    B, Lk, H, Dh = 2, 150, 2, 64
    q, k, v, dout = make(B, Lq, Lk, H, Dh, dtype, 77, packed=True)
    table = torch.full((2, H), torch.finfo(dtype).min).to(DEV, dtype)
    index = torch.randint(0, 2, (Lq, Lk), generator=torch.Generator().manual_seed(3))
    lens = [150, 67]
    got = run(q, k, v, dout, algo, bias_table=table, buckets=RelativeBuckets(index, 2).to(DEV), kv_lengths=torch.tensor(lens, device=DEV))
    want = reference(torch.zeros_like(q), k, v, Dh ** -0.5, None, lens, dout)
    want["dtable"] = bucket_sums(*want.pop("dS"), index, 2, dtype)
    for n in ("o", "dq", "dv", "dtable"):
        check(got[n], want[n], n)
    assert torch.isfinite(got["dk"]).all()


def test_operands_elsewhere_are_refused():
    q, k, v, dout = make(1, 4, 6, 2, 32, torch.bfloat16, 1, packed=True)
    plan, table = RelativeBuckets(torch.zeros(4, 6, dtype=torch.long), 1), torch.zeros(1, 2, device=DEV, dtype=torch.bfloat16)
    for args, kw in (((q, k.cpu(), v), {}), ((q, k, v), dict(kv_lengths=torch.tensor([3]))), ((q, k, v), dict(bias_table=table, buckets=plan)),
                     ((q, k, v), dict(bias_table=table.cpu(), buckets=plan.to(DEV)))):
        with pytest.raises((RuntimeError, ValueError)):
            attention(*args, **kw)


def test_backward_twice_and_retained_graphs():
    """The saved tensors are not written: a second backward over the same graph gives the same gradients, also after other
    calls have used the allocator's memory."""
    q, k, v, dout = make(2, 50, 120, 2, 64, torch.bfloat16, 41, packed=True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = attention(*leaves, kv_lengths=torch.tensor([120, 9], device=DEV))
    first = torch.autograd.grad(o, leaves, dout, retain_graph=True)
    run(*make(4, 90, 200, 2, 64, torch.bfloat16, 1, packed=True), 0, kv_lengths=torch.tensor([200, 1, 0, 30], device=DEV))
    for a, b in zip(first, torch.autograd.grad(o, leaves, dout)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,Lq,Lk,H,Dh,bias,counts", [
    (1, 100, 4097, 3, 64, False, None), (1, 100, 4097, 3, 64, True, None), (1, 40, 2305, 1, 96, False, None),
    (1, 130, 1031, 2, 128, True, None), (2, 70, 2000, 1, 64, False, [2000, 130]), (2, 48, 700, 2, 64, False, [64, 700]),
    (1, 5, 1500, 1, 88, True, [1500])])
def test_key_shares_that_do_not_divide_the_tiles(B, Lq, Lk, H, Dh, bias, counts, dtype):
    """Few rows over long memories, tile counts that the shares do not divide, counts that leave shares without any tile; the
    memory is a tensor of its own, nothing lies behind it."""
    g = torch.Generator().manual_seed(Lk)
    q, k, v, dout = [torch.randn(B, n, H, Dh, generator=g).to(DEV, dtype) for n in (Lq, Lk, Lk, Lq)]
    kw = {} if counts is None else dict(kv_lengths=torch.tensor(counts, device=DEV))
    full = None
    if bias:
        index = torch.randint(0, 30, (Lq, Lk), generator=g)
        table = torch.randn(30, H, generator=g).to(DEV, dtype)
        kw.update(bias_table=table, buckets=RelativeBuckets(index, 30).to(DEV))
        full = table.double().cpu()[index].permute(2, 0, 1)
    got = run(q, k, v, dout, 0, **kw)
    want = reference(q, k, v, Dh ** -0.5, full, counts, dout)
    dS = want.pop("dS")
    if bias:
        want["dtable"] = bucket_sums(*dS, index, 30, dtype)
    for n, w in want.items():
        check(got[n], w, n)


def shifted(t, n=1):
    """The same values, contiguous, n elements behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 16, device=t.device, dtype=t.dtype)
    out = flat[n:n + t.numel()].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_contiguous_operands_off_the_boundary(dtype):
    """Contiguous tensors at an odd storage offset, and output gradients like them, give what aligned copies give, bit for bit."""
    q, k, v, dout = [t.contiguous() for t in make(2, 40, 100, 2, 64, dtype, 4, packed=True)]
    lens = torch.tensor([100, 37], device=DEV)
    want = run(q, k, v, dout, 0, kv_lengths=lens)
    got = run(shifted(q), shifted(k, 3), shifted(v), shifted(dout), 0, kv_lengths=lens)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    w = (1 + torch.arange(64, device=DEV) / 64).to(dtype)

    def norms(q, k, dq, dk):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, w, w)]
        out = qk_norm_rope(*leaves, rope_q=rope_table(40, 64, 1), rope_k=rope_table(90, 64, 2))
        return [*out, *torch.autograd.grad(out, leaves, [dq, dk])]

    dk = torch.randn_like(k)
    for a, b in zip(norms(shifted(q), shifted(k), shifted(dout), shifted(dk, 5)), norms(q, k, dout, dk)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("batch", [None, 2])
def test_rotation_tables_off_the_boundary(batch):
    q, k, _, _ = make(2, 9, 9, 2, 80, torch.bfloat16, 4, packed=True)
    w = torch.ones(80, device=DEV)
    t = rope_table(8, 80, 3, batch)
    for a, b in zip(qk_norm_rope(q, k, w, w, rope_q=shifted(t), rope_k=shifted(t, 2)), qk_norm_rope(q, k, w, w, rope_q=t, rope_k=t)):
        assert torch.equal(a, b)


def test_head_norms_of_heads_far_apart():
    """[B, H, L, Dh] laid out, heads 2^24 elements and more apart: forward and backward as for heads side by side."""
    B, L, H, Dh = 2, 6, 3, 64
    sh = 2 ** 24 + 64
    buf = torch.empty(B * H * sh, device=DEV, dtype=torch.bfloat16)
    far = buf.as_strided((B, L, H, Dh), (H * sh, Dh, sh, 1))
    g = torch.Generator().manual_seed(2)
    far.copy_(torch.randn(B, L, H, Dh, generator=g))
    near, w, t = far.contiguous(), torch.ones(Dh, device=DEV), rope_table(L, Dh, 5)
    dy = torch.randn(B, L, H, Dh, generator=g).to(DEV, torch.bfloat16)
    dfar = torch.empty_like(buf).as_strided(far.shape, far.stride()).copy_(dy)
    outs = []
    for x, d in ((near, dy), (far, dfar)):
        x = x.detach().requires_grad_(True)
        y, none = qk_norm_rope(x, None, w, rope_q=t)
        outs.append((y, *torch.autograd.grad(y, x, d)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    want = norm_rope_reference(near, w, None, t, False, 1e-5, dy)
    check(outs[1][0], want["y"], "y")
    check(outs[1][1], want["dx"], "dx")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,L,W,off", [(1, 1, 1, 0), (5, 70, 128, 0), (5, 33, 30, 0), (3, 40, 17, 0), (4, 300, 64, 1), (700, 9, 256, 0)])
def test_padding_is_cleared(B, L, W, off, dtype):
    """Out of place and in place, units of 16, 4 and 2 bytes; rows before the counts keep their bits, NaN among them."""
    g = torch.Generator().manual_seed(L)
    flat = torch.randn(B * L * W + off, generator=g).to(DEV, dtype)
    x = flat[off:].view(B * L, W)
    x[::3] = float("nan")
    lens = torch.randint(-2, L + 3, (B,), generator=g, dtype=torch.int32)
    lens[0] = L
    live = (torch.arange(L)[None] < lens[:, None]).reshape(-1, 1).to(DEV)
    want = torch.where(live, x, torch.zeros_like(x))
    before = x.clone()
    got = K.zero_padding(x, lens.to(DEV), torch.full_like(before, 7.0))
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)) and torch.equal(x.view(torch.uint8), before.view(torch.uint8))
    assert K.zero_padding(x, lens.to(DEV), x) is x and torch.equal(x.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("algo", [0, 1])
@pytest.mark.parametrize("Lq,Lk,nb,counts", [(4, 1000, 4, None), (32, 300, 2, [300, 129]), (1, 700, 3, [128, 700]), (40, 500, 2, [500, 65])])
def test_table_gradients_do_not_see_the_rounding_of_the_output(Lq, Lk, nb, counts, algo):
    """bf16 operands, a float32 table, values with a common offset: what O's rounding to bf16 leaves in delta would add up over
    every bucket that holds much of a row.  Bound of an entry, sums over samples and rows i, and keys j of the bucket:
      * the row sums are those of numerators rounded to bf16: every probability of a row off by one factor 1 + eta, |eta| <= u
        + (Lk + 8) U, which reaches the entry through |sum_j dS_ij| alone;
      * otherwise 32-bit errors: rho of a probability (the exponential's argument, as above), Dh U |G| |V| of dP, and of
        delta = sum P dP / sum P what these and a sum of Lk leave, or for more than 32 rows and in the portable kernels (delta
        from O, less the sum of dS) eta times the rounding of O on top: u |G| |O|."""
    B, H, Dh = 2, 2, 64
    q, k, v, dout = make(B, Lq, Lk, H, Dh, torch.bfloat16, Lq + Lk, packed=False)
    v = (v.float() + 4.0).bfloat16()
    index = torch.randint(0, nb, (Lq, Lk), generator=torch.Generator().manual_seed(3))
    table = torch.randn(nb, H, generator=torch.Generator().manual_seed(4)).bfloat16().float().to(DEV)
    kw = {} if counts is None else dict(kv_lengths=torch.tensor(counts, device=DEV))
    got = run(q, k, v, dout, algo, bias_table=table, buckets=RelativeBuckets(index, nb).to(DEV), **kw)["dtable"].double().cpu()
    Q, Kk, V, G = [t.double().cpu().transpose(1, 2) for t in (q, k, v, dout)]
    dead = torch.zeros(B, 1, 1, Lk, dtype=torch.bool) if counts is None else (torch.arange(Lk)[None] >= torch.tensor(counts)[:, None])[:, None, None]
    bias = table.double().cpu()[index].permute(2, 0, 1)
    s = (Dh ** -0.5 * Q @ Kk.transpose(-1, -2) + bias).masked_fill(dead, -math.inf)
    P = s.softmax(-1)
    top = s.amax(-1, keepdim=True).abs()
    rho = (Dh + 8) * U * (Dh ** -0.5 * Q.abs() @ Kk.abs().transpose(-1, -2) + bias.abs() + top + 1.0)
    rho = 2 * rho + 2 * rho.amax(-1, keepdim=True) + 8 * U
    dP = G @ V.transpose(-1, -2)
    delta = (P * dP).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    u = half_step(torch.bfloat16)
    eta = u + (Lk + 8) * U
    edp = (Dh + 4) * U * (G.abs() @ V.abs().transpose(-1, -2))
    ed = (2 * rho * dS.abs() + P * edp).sum(-1, keepdim=True) + (Lk + 8) * U * (P * dP.abs()).sum(-1, keepdim=True)
    ed = ed + 2 * eta * u * (G.abs() * (P @ V).abs()).sum(-1, keepdim=True)
    fine = (rho * dS.abs() + P * (edp + ed)) * (1 + 1 / 16) + min(B * Lq * Lk, 4096) * U * dS.abs()
    for n in range(nb):
        m = (index == n).double()
        val = (dS * m).sum((0, 2, 3))
        bound = (eta * (dS * m).sum(-1).abs()).sum((0, 2)) + (fine * m).sum((0, 2, 3)) + 2 * U * val.abs()
        check(got[n], (val, bound), f"bucket {n}")


def dropout_call(q, k, v, dout, p, algo, **kw):
    torch.cuda.manual_seed(31)
    table = kw.pop("bias_table", None)
    old = K.set_algo(algo)
    try:
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v) + (() if table is None else (table,))]
        o = attention(*leaves[:3], bias_table=None if table is None else leaves[3], dropout=p, training=True, **kw)
        return dict(zip(("o", "dq", "dk", "dv", "dtable"), (o, *torch.autograd.grad(o, leaves, dout))))
    finally:
        K.set_algo(old)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Lq,Lk,H,Dh,bias,counts", [
    (90, 65, 2, 64, True, False), (3, 129, 2, 64, True, False), (150, 197, 1, 80, True, True), (40, 300, 2, 64, False, True),
    (1, 577, 3, 88, False, True), (197, 197, 2, 128, True, False), (300, 130, 1, 96, True, True), (33, 64, 1, 32, False, False)])
def test_dropout_beyond_one_tile_of_keys(Lq, Lk, H, Dh, bias, counts, dtype):
    """Odd key counts, key tiles behind the first, several blocks of rows and of keys, counts: the mask is read off the forward
    passes of one seed with unit vectors for 64 keys (or Dh, if fewer) at a time as the values; the gradients are those of that
    very mask, in both kernel families; 1 - p of the live probabilities are kept."""
    B, p = 2, 0.3
    q, k, v, dout = make(B, Lq, Lk, H, Dh, dtype, Lq + Lk, packed=Lq % 2 == 0)
    lens = [Lk, Lk // 2 + 1] if counts else [Lk] * B
    kw = dict(kv_lengths=torch.tensor(lens, device=DEV)) if counts else {}
    full = index = None
    if bias:
        index = torch.randint(0, 9, (Lq, Lk), generator=torch.Generator().manual_seed(2))
        kw.update(bias_table=torch.randn(9, H, generator=torch.Generator().manual_seed(3)).to(DEV, dtype), buckets=RelativeBuckets(index, 9).to(DEV))
        full = kw["bias_table"].double().cpu()[index].permute(2, 0, 1)

    def mask(algo):
        cols = []
        width = min(64, Dh)
        for k0 in range(0, Lk, width):
            unit = torch.zeros(B, Lk, H, Dh, device=DEV, dtype=dtype)
            n = min(width, Lk - k0)
            unit[:, k0:k0 + n, :, :n] = torch.eye(n, device=DEV, dtype=dtype)[None, :, None]
            o = dropout_call(q, k, unit, dout, p, algo, **kw)["o"]
            cols.append((o.detach() > 0).cpu().transpose(1, 2)[..., :n])
        return torch.cat(cols, -1)

    keep = mask(0)
    live = (torch.arange(Lk)[None] < torch.tensor(lens)[:, None])[:, None, None].expand(B, H, Lq, Lk)
    assert not keep[~live].any()
    n = int(live.sum())
    assert abs(keep[live].double().mean().item() - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n) + 1e-3
    assert torch.equal(mask(1), keep)   # both kernel families draw the same mask
    want = reference(q, k, v, Dh ** -0.5, full, lens, dout, keep=keep.double() / (1 - p))
    dS = want.pop("dS")
    if bias:
        want["dtable"] = bucket_sums(*dS, index, 9, dtype)
    for algo in (0, 1):
        got = dropout_call(q, k, v, dout, p, algo, **kw)
        for name, w in want.items():
            check(got[name], w, f"{name}, algo {algo}")


def test_every_dropout_call_draws_a_seed_of_its_own():
    q, k, v, dout = make(1, 40, 64, 1, 64, torch.bfloat16, 3, packed=True)
    torch.cuda.manual_seed(5)
    first, second = (attention(q, k, v, dropout=0.5, training=True) for _ in range(2))
    torch.cuda.manual_seed(5)
    again = attention(q, k, v, dropout=0.5, training=True)
    assert torch.equal(first, again) and not torch.equal(first, second)
    gen = torch.cuda.default_generators[torch.cuda.current_device()]
    before = gen.get_state()
    attention(q, k, v, dropout=0.5, training=False)
    attention(q, k, v, training=True)
    assert torch.equal(gen.get_state(), before)   # nothing is drawn where nothing is dropped


@pytest.mark.parametrize("algo", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,Lq,Lk,H,Dh", [(2, 1, 300, 4, 128), (2, 17, 200, 1, 128), (1, 48, 700, 2, 64), (1, 48, 700, 2, 128), (2, 9, 130, 3, 120)])
def test_wide_heads_of_few_queries_and_two_waves_that_share_keys(B, Lq, Lk, H, Dh, dtype, algo):
    """Head sizes above 96 with up to 32 queries (other buffer counts), 33 to 64 queries over enough keys to be shared out."""
    q, k, v, dout = make(B, Lq, Lk, H, Dh, dtype, Lq * 5 + Lk, packed=Dh == 64)
    index = torch.randint(0, 11, (Lq, Lk), generator=torch.Generator().manual_seed(Lk))
    table = torch.randn(11, H, generator=torch.Generator().manual_seed(Lq)).to(DEV, dtype)
    lens = [Lk - 1, 140][:B]
    got = run(q, k, v, dout, algo, bias_table=table, buckets=RelativeBuckets(index, 11).to(DEV), kv_lengths=torch.tensor(lens, device=DEV))
    want = reference(q, k, v, Dh ** -0.5, table.double().cpu()[index].permute(2, 0, 1), lens, dout)
    want["dtable"] = bucket_sums(*want.pop("dS"), index, 11, dtype)
    for n, w in want.items():
        check(got[n], w, n)


def test_dropout_is_refused_during_capture():
    """Its seed comes from the host: a replay would drop the same probabilities every time."""
    q, k, v, _ = make(1, 40, 64, 1, 64, torch.bfloat16, 3, packed=True)
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            attention(q, k, v, dropout=0.5, training=True)
    want = attention(q, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention(q, k, v, dropout=0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
