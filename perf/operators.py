"""Workloads of the attention operators: per-head normalisation with the position rotation, attention with a learned
relative position bias, and attention over memories of another (per-sample) length.

``own`` selects what ``run`` does: the plain form in elementary torch operations (32-bit arithmetic, 64 bits for the long
sums of the bias gradient, one rounding at the end), or the framework's operators as a user calls them."""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
LARGEST_WORK = 2.2e12   # operations of the largest listed case; drawn cases stay below it


def listed():
    return [
        # ---- norms of q and k for each head with the rotation in the same pass ------------------------------------------
        # one token of one sample on its way into a decoder step: nothing but latency
        dict(name="norm_rope_token", op="norm_rope", mode="fwd", dtype="bf16", norm="rms", B=1, S=1, H=12, Dh=64, prefix=0),
        # ViT-S/16 at 224 px in fp32 with LayerNorm heads and a class token: a small training step
        dict(name="norm_rope_ln_fp32", op="norm_rope", mode="train", dtype="fp32", norm="ln", B=8, S=197, H=6, Dh=64, prefix=1),
        # ViT-H/14 at 224 px, per-GPU batch 64: the head size (80) that the projection's epilogue does not take
        dict(name="norm_rope_h14", op="norm_rope", mode="train", dtype="bf16", norm="rms", B=64, S=257, H=16, Dh=80, prefix=1),
        # ViT-g/14 at 1024 px, batch 8: the longest sequence of the repository's configurations
        dict(name="norm_rope_g14_1024", op="norm_rope", mode="train", dtype="bf16", norm="rms", B=8, S=5329, H=16, Dh=88, prefix=0),
        # ---- attention with a learned relative position bias ------------------------------------------------------------
        # one small image (7 x 7 patches and a class token), inference
        dict(name="rel_bias_small", op="rel_bias", mode="fwd", dtype="bf16", B=1, gh=7, gw=7, prefix=1, H=6, Dh=64, kind="grid"),
        # ViT-B/14 at 224 px with 16 register tokens, training
        dict(name="rel_bias_b14", op="rel_bias", mode="train", dtype="bf16", B=64, gh=16, gw=16, prefix=16, H=12, Dh=64, kind="grid"),
        # ViT-S/16 at 224 px in fp32, training
        dict(name="rel_bias_s16_fp32", op="rel_bias", mode="train", dtype="fp32", B=8, gh=14, gw=14, prefix=1, H=6, Dh=64, kind="grid"),
        # ViT-g/14 at 1024 px, training, logarithmic buckets of the distance in the token sequence
        dict(name="rel_bias_g14_1024", op="rel_bias", mode="train", dtype="bf16", B=4, gh=73, gw=73, prefix=0, H=16, Dh=88, kind="log"),
        # ---- attention over memories of another length ------------------------------------------------------------------
        # serving: one query token per sample over the encoder's states of images of different sizes
        dict(name="cross_token", op="cross", mode="fwd", dtype="bf16", B=16, Lq=1, Lk=5329, H=16, Dh=88, empty=0),
        # an attentive pooling head (one learned query) over padded batches, training; one sample has no state at all
        dict(name="cross_pool", op="cross", mode="train", dtype="bf16", B=256, Lq=1, Lk=272, H=12, Dh=64, empty=1),
        # a decoder's 300 queries over the states of ViT-L/16-sized images at up to 1024 px, training
        dict(name="cross_decoder", op="cross", mode="train", dtype="bf16", B=16, Lq=300, Lk=4096, H=16, Dh=64, empty=0),
        # the same operator in fp32 at odd sizes
        dict(name="cross_decoder_fp32", op="cross", mode="train", dtype="fp32", B=4, Lq=77, Lk=577, H=12, Dh=64, empty=1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["norm_rope", "rel_bias", "cross"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        c = dict(op=op, mode=rng.choice(["fwd", "train"]), dtype=dtype, H=rng.choice([1, 2, 3, 6, 8, 12, 16]),
                 Dh=rng.choice([32, 40, 48, 64, 64, 72, 80, 88, 96, 128]))
        if op == "norm_rope":
            c.update(norm=rng.choice(["rms", "ln"]), B=_log_int(rng, 1, 256), S=_log_int(rng, 1, 5329))
            c["Dh"] = rng.choice([32, 48, 64, 80, 88, 96, 128])
            c["prefix"] = rng.randint(0, min(16, c["S"] - 1))
            if c["B"] * c["S"] * c["H"] * c["Dh"] > 8 * 5329 * 16 * 88:
                continue
        elif op == "rel_bias":
            c.update(B=_log_int(rng, 1, 64), gh=_log_int(rng, 1, 48), gw=_log_int(rng, 1, 48), prefix=rng.choice([0, 1, 5, 16]),
                     kind=rng.choice(["grid", "grid", "log"]))
        else:
            c.update(B=_log_int(rng, 1, 256), Lq=_log_int(rng, 1, 600), Lk=_log_int(rng, 1, 5329), empty=rng.randint(0, 1))
            if rng.random() < 0.4:
                c["Lq"] = 1
        if op != "norm_rope":
            scores = c["B"] * c["H"] * (_seq(c) ** 2 if op == "rel_bias" else c["Lq"] * c["Lk"])
            limit = 3.0e8 if dtype == "bf16" else 2.0e7   # the plain form holds several matrices of this many 32-bit scores
            if scores > limit or work(c)["flops"] > LARGEST_WORK:
                continue
        return c


def _seq(c):
    return c["gh"] * c["gw"] + c["prefix"]


def _lengths(c):
    """Key counts of the samples, a function of the case alone (the seed permutes them): spread over a quarter of Lk to all
    of it, the first ``empty`` samples without any key."""
    B, Lk = c["B"], c["Lk"]
    if B == 1:
        return [Lk]
    out = [max(1, Lk - (i * (Lk - Lk // 4)) // (B - 1)) for i in range(B)]
    for i in range(c["empty"]):
        out[B // 2 + i] = 0
    return out


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * std


def _rope_table(n, Dh, prefix, g):
    """[2, N, Dh] sin, cos of a line of tokens with a random phase, float32 (angles in float64)."""
    N = n - prefix
    quarter = Dh // 2
    per = 100.0 ** (2.0 * torch.arange(quarter, device=DEVICE, dtype=torch.float64) / Dh)
    pos = torch.linspace(-1, 1, max(N, 2), device=DEVICE, dtype=torch.float64)[:N]
    pos = pos + 0.1 * torch.rand(1, generator=g, device=DEVICE, dtype=torch.float64)
    ang = (2 * math.pi * pos[:, None] / per[None, :]).repeat(1, 2)
    return torch.stack([ang.sin(), ang.cos()]).float().contiguous()


def _bucket_index(c):
    """[S, S] int64 bucket numbers and their count: one per 2-D offset of two patches and three for pairs with prefix tokens
    (prefix to patch, patch to prefix, prefix to prefix), or 32 logarithmic buckets of the distance in the sequence."""
    S, prefix = _seq(c), c["prefix"]
    if c["kind"] == "log":
        pos = torch.arange(S, device=DEVICE)
        rel = pos[None, :] - pos[:, None]
        table = []   # bucket of |distance| < S, by integer arithmetic on the host
        half, exact, far = 16, 8, 128
        for d in range(S):
            b = d if d < exact else exact + int(math.floor(math.log(d / exact) / math.log(far / exact) * (half - exact) + 1e-9))
            table.append(min(b, half - 1))
        table = torch.tensor(table, device=DEVICE)
        return (table[rel.abs()] + half * (rel > 0)), 2 * half
    gh, gw = c["gh"], c["gw"]
    n_off = (2 * gh - 1) * (2 * gw - 1)
    y, x = torch.meshgrid(torch.arange(gh, device=DEVICE), torch.arange(gw, device=DEVICE), indexing="ij")
    y, x = y.reshape(-1), x.reshape(-1)
    patch = (y[:, None] - y[None, :] + gh - 1) * (2 * gw - 1) + (x[:, None] - x[None, :] + gw - 1)
    if not prefix:
        return patch, n_off
    idx = torch.empty((S, S), dtype=torch.int64, device=DEVICE)
    idx[prefix:, prefix:] = patch
    idx[:prefix, prefix:] = n_off
    idx[prefix:, :prefix] = n_off + 1
    idx[:prefix, :prefix] = n_off + 2
    return idx, n_off + 3


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    train = c["mode"] == "train"
    H, Dh = c["H"], c["Dh"]
    s = dict(case=dict(c))

    if own:
        from vit_amd.attention import attention, qk_norm_rope

        s["call"] = qk_norm_rope if c["op"] == "norm_rope" else attention

    def leaf(t):
        return t.detach().requires_grad_(train)

    if c["op"] == "norm_rope":
        B, S = c["B"], c["S"]
        qkv = _randn(g, B, S, 3, H, Dh).to(dt)   # the packed projection: q and k are views of it
        s["q"], s["k"] = leaf(qkv[:, :, 0]), leaf(qkv[:, :, 1])
        ln = c["norm"] == "ln"
        s["qw"], s["kw"] = [leaf((1.0 + _randn(g, Dh, std=0.2)).to(dt)) for _ in range(2)]
        s["qb"], s["kb"] = [leaf(_randn(g, Dh, std=0.2).to(dt)) if ln else None for _ in range(2)]
        s["rope"] = _rope_table(S, Dh, c["prefix"], g)
        if train:
            s["dq"], s["dk"] = [_randn(g, B, S, H, Dh).to(dt) for _ in range(2)]
        return s
    if c["op"] == "rel_bias":
        B, S = c["B"], _seq(c)
        qkv = _randn(g, B, S, 3, H, Dh).to(dt)
        s["q"], s["k"], s["v"] = [leaf(qkv[:, :, i]) for i in range(3)]
        idx, nb = _bucket_index(c)
        s["index"], s["num_buckets"] = idx.to(torch.int32), nb
        s["table"] = leaf(_randn(g, nb, H, std=0.7).to(dt))
        if train and not own:   # pairs sorted by bucket, and where each bucket ends: kept with the index
            flat, s["order"] = torch.sort(s["index"].reshape(-1), stable=True)
            s["ends"] = torch.searchsorted(flat, torch.arange(nb + 1, device=DEVICE, dtype=torch.int32))
        if own:   # the plan a model builds once from its grid
            from vit_amd.pos_enc import RelativeBuckets

            s["buckets"] = RelativeBuckets(s["index"], nb)
        Lq = S
    else:
        B, Lq, Lk = c["B"], c["Lq"], c["Lk"]
        s["q"] = leaf(_randn(g, B, Lq, H, Dh).to(dt))
        kv = _randn(g, B, Lk, 2, H, Dh).to(dt)   # the packed key | value projection of the memory
        s["k"], s["v"] = leaf(kv[:, :, 0]), leaf(kv[:, :, 1])
        perm = torch.randperm(B, generator=g, device=DEVICE)
        s["lengths"] = torch.tensor(_lengths(c), device=DEVICE, dtype=torch.int32)[perm].contiguous()
    if train:
        s["do"] = _randn(g, B, Lq, H, Dh).to(dt)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    c = s["case"]
    call = s["call"]
    train = c["mode"] == "train"
    if c["op"] == "norm_rope":
        ln = c["norm"] == "ln"
        q, k = call(s["q"], s["k"], s["qw"], s["kw"], s["qb"], s["kb"], rope_q=s["rope"], rope_k=s["rope"], eps=EPS,
                    use_layer_norm=ln)
        out = dict(q=q, k=k)
        if train:
            names = ["q", "k", "qw", "kw"] + (["qb", "kb"] if ln else [])
            grads = torch.autograd.grad([q, k], [s[n] for n in names], [s["dq"], s["dk"]])
            out = dict(q=q.detach(), k=k.detach(), **{"d" + n: t for n, t in zip(names, grads)})
        return out
    if c["op"] == "rel_bias":
        o = call(s["q"], s["k"], s["v"], bias_table=s["table"], buckets=s["buckets"])
        names = ["q", "k", "v", "table"]
    else:
        o = call(s["q"], s["k"], s["v"], kv_lengths=s["lengths"])
        names = ["q", "k", "v"]
    if not train:
        return dict(o=o)
    grads = torch.autograd.grad(o, [s[n] for n in names], s["do"])
    return dict(o=o.detach(), **{"d" + n: t for n, t in zip(names, grads)})


def _rot_half(x):
    h = x.shape[-1] // 2
    return torch.cat([-x[..., h:], x[..., :h]], dim=-1)


def _plain_norm_rope(x, w, b, table, prefix, ln):
    """(y, xhat, rstd): normalised heads, scaled, rotated behind the prefix."""
    xf = x.detach().float()
    xc = xf - xf.mean(-1, keepdim=True) if ln else xf
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xhat = xc * rstd
    n = xhat * w.detach().float()
    if b is not None:
        n = n + b.detach().float()
    sin, cos = table[0][None, :, None], table[1][None, :, None]
    r = n[:, prefix:]
    return torch.cat([n[:, :prefix], r * cos + _rot_half(r) * sin], dim=1), xhat, rstd


def _plain_norm_rope_bwd(dy, xhat, rstd, w, table, prefix, ln):
    g = dy.float()
    sin, cos = table[0][None, :, None], table[1][None, :, None]
    r = g[:, prefix:]
    t = r * sin
    h = t.shape[-1] // 2
    dn = torch.cat([g[:, :prefix], r * cos + torch.cat([t[..., h:], -t[..., :h]], dim=-1)], dim=1)
    # the sums over all rows in 64 bits
    dw = (dn * xhat).double().sum(dim=(0, 1, 2))
    db = dn.double().sum(dim=(0, 1, 2))
    u = dn * w.detach().float()
    dx = u - xhat * (u * xhat).mean(-1, keepdim=True)
    if ln:
        dx = dx - u.mean(-1, keepdim=True)
    return dx * rstd, dw, db


def _run_plain(s):
    c = s["case"]
    train = c["mode"] == "train"
    dt = DTYPES[c["dtype"]]
    with torch.no_grad():
        if c["op"] == "norm_rope":
            ln = c["norm"] == "ln"
            out, bwd = {}, {}
            for n in ("q", "k"):
                y, xhat, rstd = _plain_norm_rope(s[n], s[n + "w"], s[n + "b"], s["rope"], c["prefix"], ln)
                out[n] = y.to(dt)
                if train:
                    dx, dw, db = _plain_norm_rope_bwd(s["d" + n], xhat, rstd, s[n + "w"], s["rope"], c["prefix"], ln)
                    bwd["d" + n], bwd["d" + n + "w"], bwd["d" + n + "b"] = dx.to(dt), dw.to(dt), db.to(dt)
            if not train:
                return out
            names = ["q", "k", "qw", "kw"] + (["qb", "kb"] if ln else [])
            return dict(out, **{"d" + n: bwd["d" + n] for n in names})
        scale = c["Dh"] ** -0.5
        q, k, v = [s[n].detach().float().transpose(1, 2).contiguous() for n in ("q", "k", "v")]   # [B, H, L, Dh]
        sc = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
        if c["op"] == "rel_bias":
            bias = s["table"].detach().float()[s["index"].long()]            # [S, S, H]
            sc = sc + bias.permute(2, 0, 1)[None]
        else:
            dead = torch.arange(c["Lk"], device=DEVICE)[None, :] >= s["lengths"][:, None]
            v = v.masked_fill(dead[:, None, :, None], 0.0)
            sc = sc.masked_fill(dead[:, None, None, :], -math.inf)
        m = sc.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, torch.zeros_like(m), m)
        p = torch.exp(sc - m)
        del sc
        l = p.sum(-1, keepdim=True)
        p = p / torch.where(l == 0, torch.ones_like(l), l)
        o = torch.matmul(p, v)
        out = dict(o=o.transpose(1, 2).to(dt).contiguous())
        if not train:
            return out
        do = s["do"].float().transpose(1, 2).contiguous()
        dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
        delta = (do * o).sum(-1, keepdim=True)
        ds = p * (torch.matmul(do, v.transpose(-1, -2).contiguous()) - delta)
        del p
        if c["op"] == "cross":
            k = k.masked_fill(dead[:, None, :, None], 0.0)
        out["dq"] = (torch.matmul(ds, k) * scale).transpose(1, 2).to(dt).contiguous()
        out["dk"] = (torch.matmul(ds.transpose(-1, -2).contiguous(), q) * scale).transpose(1, 2).to(dt).contiguous()
        out["dv"] = dv.transpose(1, 2).to(dt).contiguous()
        if c["op"] == "rel_bias":
            S = _seq(c)
            # pairs in the order of their buckets: a bucket's sum is the difference of two running sums (64 bits)
            dbias = ds.sum(0).reshape(c["H"], S * S)
            del ds
            sums = []
            for h in range(c["H"]):
                run_sum = torch.cumsum(dbias[h][s["order"]].double(), 0)
                sums.append(torch.cat([run_sum.new_zeros(1), run_sum])[s["ends"]].diff())
            out["dtable"] = torch.stack(sums, dim=1).to(dt)
        return out


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(c, seed)
    train = c["mode"] == "train"
    D = torch.float64
    if c["op"] == "norm_rope":
        out, grads = {}, {}
        ln = c["norm"] == "ln"
        for n in ("q", "k"):
            x = s[n].detach().to(D).requires_grad_(train)
            w = s[n + "w"].detach().to(D).requires_grad_(train)
            b = s[n + "b"].detach().to(D).requires_grad_(train) if ln else None
            mean = x.mean(-1, keepdim=True) if ln else 0.0
            z = (x - mean) / ((x - mean).square().mean(-1, keepdim=True) + EPS).sqrt() * w
            z = z + b if ln else z
            a, e = z[:, :, :, :c["Dh"] // 2], z[:, :, :, c["Dh"] // 2:]
            sin = torch.zeros((c["S"], c["Dh"]), dtype=D, device=DEVICE)
            cos = torch.ones((c["S"], c["Dh"]), dtype=D, device=DEVICE)
            sin[c["prefix"]:], cos[c["prefix"]:] = s["rope"][0].to(D), s["rope"][1].to(D)
            sin, cos = sin[None, :, None], cos[None, :, None]
            h = c["Dh"] // 2
            y = torch.cat([a * cos[..., :h] - e * sin[..., :h], e * cos[..., h:] + a * sin[..., h:]], dim=-1)
            out[n] = y.detach()
            if train:
                leaves = [x, w] + ([b] if ln else [])
                gs = torch.autograd.grad(y, leaves, s["d" + n].to(D))
                grads["d" + n], grads["d" + n + "w"] = gs[0], gs[1]
                if ln:
                    grads["d" + n + "b"] = gs[2]
        if not train:
            return out
        names = ["q", "k", "qw", "kw"] + (["qb", "kb"] if ln else [])
        return dict(out, **{"d" + n: grads["d" + n] for n in names})

    q, k, v = [s[n].detach() for n in ("q", "k", "v")]
    B, Lq, H, Dh = q.shape
    Lk = k.shape[1]
    names = ["o"] + (["dq", "dk", "dv"] if train else [])
    shapes = dict(o=q.shape, dq=q.shape, dk=k.shape, dv=v.shape)
    out = {n: torch.zeros(shapes[n], dtype=D, device=DEVICE) for n in names}
    rel = c["op"] == "rel_bias"
    lens = [Lk] * B if rel else s["lengths"].tolist()
    if rel:
        index = s["index"].long()
        if train:
            flat = index.reshape(-1).cpu().numpy()
            dtab = torch.zeros((s["num_buckets"], H), dtype=D, device=DEVICE)
    # sample by sample (or head by head where one sample's scores are large)
    step = H if H * Lq * Lk <= 5e7 else 1
    for h0 in range(0, H, step):
        hs = slice(h0, h0 + step)
        if rel:
            bias = s["table"].detach().to(D)[:, hs].t()[:, index.reshape(-1)].reshape(-1, Lq, Lk)
            dbias = torch.zeros_like(bias) if train else None
        for b in range(B):
            n = int(lens[b])
            if n == 0:
                continue
            qb = q[b, :, hs].to(D).permute(1, 0, 2).contiguous()
            kb, vb = [t[b, :n, hs].to(D).permute(1, 0, 2).contiguous() for t in (k, v)]
            z = torch.bmm(qb, kb.transpose(1, 2).contiguous()) / math.sqrt(Dh)
            if rel:
                z += bias
            p = (z - z.amax(2, keepdim=True)).exp_()
            p /= p.sum(2, keepdim=True)
            ob = torch.bmm(p, vb)
            out["o"][b, :, hs] = ob.permute(1, 0, 2)
            if train:
                gb = s["do"][b, :, hs].to(D).permute(1, 0, 2).contiguous()
                out["dv"][b, :n, hs] = torch.bmm(p.transpose(1, 2).contiguous(), gb).permute(1, 0, 2)
                dz = torch.bmm(gb, vb.transpose(1, 2).contiguous())
                dz -= (gb * ob).sum(2, keepdim=True)
                dz *= p
                out["dq"][b, :, hs] = torch.bmm(dz, kb).permute(1, 0, 2) / math.sqrt(Dh)
                out["dk"][b, :n, hs] = torch.bmm(dz.transpose(1, 2).contiguous(), qb).permute(1, 0, 2) / math.sqrt(Dh)
                if rel:
                    dbias += dz
        if rel and train:
            for i, h in enumerate(range(H)[hs]):
                sums = np.bincount(flat, weights=dbias[i].reshape(-1).cpu().numpy(), minlength=s["num_buckets"])
                dtab[:, h] = torch.from_numpy(sums).to(DEVICE)
    if rel and train:
        out["dtable"] = dtab
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    c = case
    es = 2 if c["dtype"] == "bf16" else 4
    train = c["mode"] == "train"
    H, Dh = c["H"], c["Dh"]
    if c["op"] == "norm_rope":
        n = 2 * c["B"] * c["S"] * H * Dh
        table = 2 * (c["S"] - c["prefix"]) * Dh * 4
        # forward: read x, write y; backward: read dy and x, write dx
        return dict(bytes=float(n * es * (5 if train else 2) + table * (2 if train else 1)), flops=float(n * (25 if train else 9)))
    if c["op"] == "rel_bias":
        B, S = c["B"], _seq(c)
        x = B * S * H * Dh
        pairs = B * H * S * S
        nb = 32 if c["kind"] == "log" else (2 * c["gh"] - 1) * (2 * c["gw"] - 1) + (3 if c["prefix"] else 0)
        return dict(bytes=float(x * es * (8 if train else 4) + nb * H * es * (2 if train else 1) + S * S * 4),
                    flops=float(pairs * Dh * (14 if train else 4)))
    B, Lq, Lk = c["B"], c["Lq"], c["Lk"]
    keys = sum(_lengths(c))
    x, m, whole = B * Lq * H * Dh, keys * H * Dh, B * Lk * H * Dh
    # forward: read q and the live keys and values, write o; training adds do, dq and the whole dk, dv
    return dict(bytes=float(es * (2 * x + 2 * m + (2 * x + 2 * whole if train else 0)) + 4 * B),
                flops=float(Lq * keys * H * Dh * (14 if train else 4)))
