"""The relative position bias, the key counts, the per-head normalisation pass and projected memories inside the layers:
against the same layers without padding, against plain arithmetic, and together."""
import copy
import math

import pytest
import torch

from vit_amd import AttentivePoolHead, RelativeBuckets, ViTConfig
from vit_amd.attention import AttentivePool, CrossAttention, SelfAttention
from vit_amd.transformer import CrossAttentionTransformer, TransformerDecoderLayer

pytestmark = pytest.mark.gpu

DEV = "cuda"
MODES = [(torch.float32, False), (torch.bfloat16, False), (torch.float32, True)]
MODE_IDS = ["fp32", "bf16", "autocast"]


def tol(dtype, autocast):
    """Two runs of the same layer over differently shaped launches: sums of D <= 160 products in another order (fp32), and
    for bf16 a handful of roundings (projection, heads, probabilities, output: 8 half steps of 2^-8) of the largest value."""
    return 1e-4 if dtype == torch.float32 and not autocast else 8 * 2.0 ** -8


def close(a, b, t, msg=""):
    a, b = a.detach().double(), b.detach().double()
    lim = t * max(b.abs().max().item(), 1e-6)
    assert torch.isfinite(a).all(), msg
    assert (a - b).abs().max().item() <= lim, f"{msg}: {(a - b).abs().max().item():.3e} > {lim:.3e}"


def randomize(module, seed=0):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in module.parameters():
            p.copy_((0.1 * torch.randn(p.shape, generator=g) + (1.0 if p.dim() == 1 and "norm" in str(p.shape) else 0.0)).to(p))
        for n, p in module.named_parameters():
            if n.endswith("norm.weight"):
                p.add_(1.0)
    return module


@pytest.mark.parametrize("dtype,autocast", MODES, ids=MODE_IDS)
@pytest.mark.parametrize("Dh,qk_norm,norm", [(64, False, "rmsnorm"), (80, True, "rmsnorm"), (32, True, "layernorm")])
def test_padded_batch_equals_each_sample_alone(dtype, autocast, Dh, qk_norm, norm, monkeypatch):
    """A decoder layer with self-attention under a relative bias and cross-attention to padded memories: the outputs, the
    input gradients and the weights' gradients equal the sum over the samples run alone without padding."""
    D, H, Lq, Lk = 2 * Dh, 2, 9, 70
    lens = [70, 1, 33]
    layer = randomize(TransformerDecoderLayer(D, 2 * D, H, 0.0, 0.0, norm_type=norm, qk_normalization=qk_norm, device=DEV,
                                              dtype=dtype, activation="silu", relative_buckets=25)).train()
    g = torch.Generator().manual_seed(1)
    x, kv = torch.randn(3, Lq, D, generator=g).to(DEV, dtype), torch.randn(3, Lk, D, generator=g).to(DEV, dtype)
    dy = torch.randn(3, Lq, D, generator=g).to(DEV, dtype)
    plan = RelativeBuckets.grid((3, 3), device=DEV)
    for b, n in enumerate(lens):
        kv[b, n:] = 100.0   # padding: finite (it passes the projection), far from anything that would go unnoticed

    def go(x, kv, dy, lengths):
        layer.zero_grad()
        x, kv = x.clone().requires_grad_(True), kv.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            y = layer(x, kv, kv_lengths=lengths, buckets=plan)
        y.backward(dy.to(y.dtype))
        return y, x.grad, kv.grad, {n: p.grad.clone() for n, p in layer.named_parameters()}

    largest = [0.0]   # entry of the gradient of the normalised keys, over all calls
    from vit_amd import kernels as K
    inner = K.qk_norm_rope_bwd
    monkeypatch.setattr(K, "qk_norm_rope_bwd", lambda xs, gs, *a, **kw: (
        largest.__setitem__(0, max(largest[0], gs[1].float().abs().max().item())), inner(xs, gs, *a, **kw))[1])
    y, dx, dkv, dw = go(x, kv, dy, torch.tensor(lens, device=DEV))
    t = tol(dtype, autocast)
    total = None
    for b, n in enumerate(lens):
        y1, dx1, dkv1, dw1 = go(x[b:b + 1], kv[b:b + 1, :n], dy[b:b + 1], None)
        close(y[b:b + 1], y1, t, "y")
        close(dx[b:b + 1], dx1, 2 * t, "dx")
        close(dkv[b:b + 1, :n], dkv1, 2 * t, "dkv")
        assert not dkv[b, n:].any()
        total = dw1 if total is None else {k: total[k].double() + dw1[k].double() for k in dw1}
    for k in dw:
        if k.endswith("k_norm.bias"):
            # Without a rotation a bias b on every key adds q b to all scores of a row, which the softmax does not see: this
            # gradient is zero (a row of dS sums to zero).  What is left on both sides is the rounding of the summed entries
            # of dk, each at most t of the largest: R = 3 samples x 2 heads x (9 or 70) rows of them.
            rows = 3 * H * (Lq if k.startswith("self") else Lk)
            assert dw[k].abs().max().item() <= rows * t * largest[0] and total[k].abs().max().item() <= rows * t * largest[0]
            continue
        close(dw[k], total[k], 2 * t, k)


@pytest.mark.parametrize("dtype,autocast", MODES, ids=MODE_IDS)
@pytest.mark.parametrize("layer_type", [TransformerDecoderLayer, CrossAttentionTransformer])
def test_projected_memory_equals_the_states(dtype, autocast, layer_type):
    """Single decoder tokens over a memory projected once, with rotation, per-head normalisation and key counts."""
    D, H, Lk = 160, 2, 90
    layer = randomize(layer_type(D, 2 * D, H, 0.0, 0.0, qk_normalization=True, device=DEV, dtype=dtype, activation="silu",
                                 layer_scale=0.5)).eval()
    g = torch.Generator().manual_seed(2)
    kv = torch.randn(2, Lk, D, generator=g).to(DEV, dtype)
    lens = torch.tensor([90, 41], device=DEV)
    ang = torch.rand(Lk, 80, generator=g) * 6
    rope = torch.stack([ang.sin(), ang.cos()]).to(DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        memory = layer.cross_attention.project_kv(kv, rope_k=rope, kv_lengths=lens)
        for step in range(3):
            x = torch.randn(2, 1, D, generator=g).to(DEV, dtype)
            rq = rope[:, step:step + 1].contiguous()
            want = layer(x, kv, rope_q=rq, rope_k=rope, kv_lengths=lens)
            assert torch.equal(layer(x, memory, rope_q=rq), want)
        want = layer.cross_attention(x, kv, rope_q=rq, rope_k=rope, kv_lengths=lens)
        assert torch.equal(layer.cross_attention(x, memory, rope_q=rq), want)


@pytest.mark.parametrize("dtype,autocast", MODES, ids=MODE_IDS)
def test_pooling_over_padded_tokens(dtype, autocast):
    D, H, L = 128, 2, 300
    lens = [300, 0, 17, 299]
    for nq in (1, 3):
        pool = randomize(AttentivePool(D, H, num_queries=nq, device=DEV, dtype=dtype))
        x = torch.randn(4, L, D, generator=torch.Generator().manual_seed(3)).to(DEV, dtype)
        xg = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            y = pool(xg, torch.tensor(lens, device=DEV))
            y.float().square().sum().backward()
            assert y.shape == ((4, D) if nq == 1 else (4, nq, D))
            for b, n in enumerate(lens):
                assert not xg.grad[b, n:].any()
                if n:
                    close(y[b:b + 1], pool(x[b:b + 1, :n].contiguous()), tol(dtype, autocast), "pool")
                else:   # no token: the projection of zeros
                    bias = pool.cross_attention.out_proj.bias
                    close(y[b].reshape(-1, D), bias.expand(nq, D), tol(dtype, autocast), "empty")
    head = AttentivePoolHead(D, 10, H, device=DEV, dtype=dtype)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        assert head(x, torch.tensor(lens, device=DEV)).shape == (4, 10)


@pytest.mark.parametrize("dtype,autocast", MODES, ids=MODE_IDS)
@pytest.mark.parametrize("Dh", [64, 80])
def test_self_attention_with_relative_bias_matches_plain_arithmetic(dtype, autocast, Dh):
    """The whole sub-layer, with q / k normalisation and the rotation, against torch operations in 64 bits and autograd."""
    H, S, B = 2, 21, 3
    D = H * Dh
    att = randomize(SelfAttention(D, H, 0.0, 0.0, qk_normalization=True, device=DEV, dtype=dtype, relative_buckets=35 + 3))
    plan = RelativeBuckets.grid((4, 3), 9, device=DEV, table_dims=(4, 3))
    g = torch.Generator().manual_seed(4)
    x = torch.randn(B, S, D, generator=g).to(DEV, dtype)
    dy = torch.randn(B, S, D, generator=g).to(DEV, dtype)
    ang = torch.rand(S - 9, Dh, generator=g) * 6
    rope = torch.stack([ang.sin(), ang.cos()]).to(DEV)

    ref = copy.deepcopy(att).double().cpu()
    xr = x.double().cpu().requires_grad_(True)
    rms = lambda t, w: t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w
    qkv = torch.nn.functional.linear(rms(xr, ref.norm.weight), ref.qkv_proj.weight, ref.qkv_proj.bias).view(B, S, 3, H, Dh)
    q, k, v = (t.transpose(1, 2) for t in qkv.unbind(2))
    q, k = rms(q, ref.q_norm.weight), rms(k, ref.k_norm.weight)
    sin, cos = rope.double().cpu()

    def rot(t):
        p, r = t[:, :, :9], t[:, :, 9:]
        h = Dh // 2
        return torch.cat([p, r * cos + torch.cat([-r[..., h:], r[..., :h]], -1) * sin], 2)

    index = (plan.index16.cpu().long() & 0xFFFF)
    s = rot(q) @ rot(k).transpose(-1, -2) * Dh ** -0.5 + ref.relative_bias[index].permute(2, 0, 1)
    o = (s.softmax(-1) @ v).transpose(1, 2).reshape(B, S, D)
    yr = torch.nn.functional.linear(o, ref.out_proj.weight, ref.out_proj.bias)
    yr.backward(dy.double().cpu())

    xg = x.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        y = att(xg, rope=rope, buckets=plan)
    y.backward(dy.to(y.dtype))
    # norm, projection, heads, rotation, probabilities, output and their counterparts backward: 20 half steps of the largest
    t = 1e-4 if tol(dtype, autocast) == 1e-4 else 20 * 2.0 ** -8
    close(y.cpu(), yr, t, "y")
    close(xg.grad.cpu(), xr.grad, t, "dx")
    for (n, p), (_, pr) in zip(att.named_parameters(), ref.named_parameters()):
        assert p.grad.dtype == p.dtype, n
        close(p.grad.cpu(), pr.grad, t, n)


@pytest.mark.parametrize("ckpt", [False, True])
def test_relative_vit_trains_and_learns_from_its_tables(ckpt):
    """A ViT with pos_enc "relative": gradients of tables, weights and inputs against the same model in fp32, other token
    grids, drop-path and dropout run, and checkpointing replays the same gradients."""
    kw = dict(in_channels=3, patch_size=(8, 8), img_size=(40, 32), depth=2, hidden_size=128, ffn_hidden_size=256,
              num_attention_heads=2, num_register_tokens=2, num_cls_tokens=1, pos_enc="relative", dtype=torch.float32,
              activation="swiglu", activation_checkpointing=ckpt)
    model = randomize(ViTConfig(**kw, hidden_dropout=0.0, attention_dropout=0.0).instantiate(device=DEV)).train()
    x = torch.randn(3, 3, 40, 32, generator=torch.Generator().manual_seed(5)).to(DEV)

    def grads(autocast):
        model.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            model(x).dense_features.float().square().mean().backward()
        return {n: p.grad.clone() for n, p in model.named_parameters()}

    full, low = grads(False), grads(True)
    for n in full:
        assert full[n].abs().max() > 0 or "norm" in n, n
        close(low[n], full[n], 40 * 2.0 ** -8, n)
    again = grads(False)
    assert all(torch.equal(full[n], again[n]) for n in full)
    small = model(torch.randn(2, 3, 24, 32, device=DEV)).visual_tokens
    assert small.shape == (2, 12, 128) and torch.isfinite(small).all()
    noisy = randomize(ViTConfig(**kw, hidden_dropout=0.1, attention_dropout=0.1, drop_path_rate=0.4).instantiate(device=DEV)).train()
    noisy(x).dense_features.square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in noisy.parameters())
    assert noisy.blocks[0].self_attention.relative_bias.grad.abs().max() > 0


def test_drop_path_picks_the_counts_of_its_samples():
    torch.manual_seed(3)
    D, H = 64, 2
    layer = randomize(CrossAttentionTransformer(D, 128, H, 0.0, 0.0, drop_path_rate=0.5, device=DEV, dtype=torch.float32,
                                                activation="silu")).train()
    x, kv = torch.randn(6, 4, D, device=DEV), torch.randn(6, 30, D, device=DEV)
    lens = torch.tensor([0, 1, 7, 30, 16, 29], device=DEV)
    for b in range(6):
        kv[b, lens[b]:] = 50.0
    kvg = kv.clone().requires_grad_(True)
    layer(x, kvg, kv_lengths=lens).square().sum().backward()
    took_part = [bool(kvg.grad[b].any()) for b in range(6)]
    assert 0 < sum(took_part) <= 3
    for b in range(6):
        assert not kvg.grad[b, lens[b]:].any()


def test_head_norm_pass_keeps_the_results_of_the_separate_passes(monkeypatch):
    """Head size 80 in the layers: the one-pass form against norm, copy and rotation as passes of their own.  The sums run
    in another order, so a rounded value may move by one step of bf16 (2^-7); everything else is the same arithmetic."""
    from vit_amd import kernels as K

    D, H, S = 160, 2, 50
    att = randomize(SelfAttention(D, H, 0.0, 0.0, qk_normalization=True, device=DEV, dtype=torch.bfloat16))
    x = torch.randn(4, S, D, generator=torch.Generator().manual_seed(6)).to(DEV, torch.bfloat16)
    ang = torch.rand(S - 1, 80, generator=torch.Generator().manual_seed(7)) * 6
    rope = torch.stack([ang.sin(), ang.cos()]).to(DEV, torch.bfloat16)

    def go():
        att.zero_grad()
        xg = x.clone().requires_grad_(True)
        y = att(xg, rope=rope)
        y.float().square().mean().backward()
        return [y, xg.grad] + [p.grad.clone() for p in att.parameters()]

    one = go()
    monkeypatch.setattr(K, "can_qk_norm_rope", lambda *a: False)
    for a, b in zip(one, go()):
        close(a, b, 2.0 ** -7, "passes")


def test_training_step_of_a_decoder_captures_into_a_graph():
    D, H = 128, 2
    layer = randomize(TransformerDecoderLayer(D, 256, H, 0.0, 0.0, qk_normalization=True, device=DEV, dtype=torch.bfloat16,
                                              activation="silu", relative_buckets=25)).train()
    plan = RelativeBuckets.grid((3, 3), device=DEV)
    x, kv = torch.randn(2, 9, D, device=DEV).bfloat16(), torch.randn(2, 700, D, device=DEV).bfloat16()
    lens = torch.tensor([700, 300], device=DEV, dtype=torch.int32)
    params = list(layer.parameters())

    def step():
        return [t.detach() for t in torch.autograd.grad(layer(x, kv, kv_lengths=lens, buckets=plan).float().square().mean(), params)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for rep in range(3):
        x.copy_(torch.randn_like(x))
        kv.copy_(torch.randn_like(kv))
        lens.copy_(torch.tensor([700 - rep, rep], device=DEV))
        want = [t.clone() for t in step()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), rep


def test_layers_take_rotation_tables_off_the_boundary():
    """A contiguous float32 table one element behind a boundary, through the layers that normalise and rotate in one pass."""
    D, H, S = 160, 2, 11
    g = torch.Generator().manual_seed(1)
    ang = torch.rand(S, 80, generator=g) * 6
    rope = torch.stack([ang.sin(), ang.cos()]).to(DEV)
    off = torch.empty(rope.numel() + 1, device=DEV)[1:].view(rope.shape).copy_(rope)
    assert off.is_contiguous() and off.data_ptr() % 16
    layer = randomize(TransformerDecoderLayer(D, 2 * D, H, 0.0, 0.0, qk_normalization=True, device=DEV, dtype=torch.bfloat16,
                                              activation="silu")).train()
    x, kv = torch.randn(2, S, D, generator=g).to(DEV, torch.bfloat16), torch.randn(2, S, D, generator=g).to(DEV, torch.bfloat16)

    def go(rope):
        layer.zero_grad()
        y = layer(x, kv, rope_q=rope, rope_k=rope)
        y.float().square().mean().backward()
        return [y] + [p.grad.clone() for p in layer.parameters()]

    for a, b in zip(go(off), go(rope)):
        assert torch.equal(a, b)


BAD = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("dtype,autocast", MODES, ids=MODE_IDS)
@pytest.mark.parametrize("Dh,qk_norm,norm", [(64, False, "rmsnorm"), (80, True, "rmsnorm"), (32, True, "layernorm"), (12, True, "rmsnorm")])
def test_training_does_not_see_what_padding_holds(dtype, autocast, Dh, qk_norm, norm):
    """Padded rows of a memory that hold NaN and infinities: outputs, the weights' gradients and those of the inputs are the
    ones of a memory padded with ones, bit for bit, with and without drop-path's choice of samples; the memory is not written."""
    D, H, Lq, Lk, B = 2 * Dh, 2, 9, 70, 6
    lens = [70, 1, 33, 0, 64, 69]
    g = torch.Generator().manual_seed(1)
    x, kv = torch.randn(B, Lq, D, generator=g).to(DEV, dtype), torch.randn(B, Lk, D, generator=g).to(DEV, dtype)
    ones, bad = kv.clone(), kv.clone()
    for b, n in enumerate(lens):
        ones[b, n:] = 1.0
        bad[b, n:] = BAD[b % 3]
    for drop in (0.0, 0.5):
        layer = randomize(TransformerDecoderLayer(D, 2 * D, H, 0.0, 0.0, norm_type=norm, qk_normalization=qk_norm, device=DEV, dtype=dtype,
                                                  activation="silu", drop_path_rate=drop)).train()

        def go(kv):
            layer.zero_grad()
            torch.manual_seed(7)
            xg, kvg = x.clone().requires_grad_(True), kv.clone().requires_grad_(True)
            before = kvg.detach().clone()
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
                y = layer(xg, kvg, kv_lengths=torch.tensor(lens, device=DEV))
            y.float().square().mean().backward()
            assert torch.equal(kvg.detach().view(torch.uint8), before.view(torch.uint8))
            return [y, xg.grad, kvg.grad] + [p.grad.clone() for p in layer.parameters()]

        for i, (a, b) in enumerate(zip(go(bad), go(ones))):
            assert torch.isfinite(a).all() and torch.equal(a, b), (drop, i)


@pytest.mark.parametrize("frozen", [False, True])
def test_pooling_trains_on_padding_that_holds_anything(frozen):
    """The pooling head over states without a gradient of their own (a frozen encoder's) and with one."""
    D, H, L = 128, 2, 300
    lens = torch.tensor([300, 0, 17, 299], device=DEV)
    head = randomize(AttentivePoolHead(D, 10, H, device=DEV, dtype=torch.bfloat16)).train()
    x = torch.randn(4, L, D, generator=torch.Generator().manual_seed(3)).to(DEV, torch.bfloat16)
    grads = []
    for fill in (1.0, float("nan")):
        for b in range(4):
            x[b, int(lens[b]):] = fill
        head.zero_grad()
        xg = x.clone().requires_grad_(not frozen)
        head(xg, lens).float().square().sum().backward()
        grads.append([p.grad.clone() for p in head.parameters()] + ([] if frozen else [xg.grad]))
    for a, b in zip(*grads):
        assert torch.isfinite(b).all() and torch.equal(a, b)


def relative_vit(**kw):
    cfg = dict(in_channels=3, patch_size=(8, 8), img_size=(96, 96), depth=1, hidden_size=128, ffn_hidden_size=256, num_attention_heads=2,
               pos_enc="relative", dtype=torch.bfloat16, hidden_dropout=0.0, attention_dropout=0.0)
    return ViTConfig(**{**cfg, **kw}).instantiate(device=DEV).eval()


def test_dropped_plans_keep_their_memory_until_their_streams_are_through():
    """A plan made on one stream and used on another, dropped by eight newer grids while that work is still waiting: what is
    allocated meanwhile does not get its memory; once the work is done, it does."""
    model = relative_vit()
    model.prepare_buckets((12, 12))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        model(torch.randn(1, 3, 96, 96, device=DEV, dtype=torch.bfloat16))
        torch.cuda._sleep(400_000_000)   # some tenths of a second
    plan = model.prepare_buckets((12, 12))
    place = {t.data_ptr(): t.numel() * t.element_size() for t in (plan.index16, plan.order)}
    del plan
    busy = not side.query()
    for n in range(1, 9):
        model.prepare_buckets((1, n))
    assert ((12, 12), model.cls_tokens.device) not in model._bucket_plans
    held = [torch.empty(16384, device=DEV, dtype=torch.uint8) for _ in range(2000)]
    still = not side.query()
    if busy and still:
        for t in held:
            assert not any(at < t.data_ptr() + t.numel() and t.data_ptr() < at + n for at, n in place.items())
    torch.cuda.synchronize()
    assert busy and still, "the side stream was through too early to tell"


def test_a_plan_is_not_made_during_capture():
    model = relative_vit()
    x = torch.randn(2, 3, 64, 96, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        model(torch.randn(2, 3, 96, 96, device=DEV, dtype=torch.bfloat16))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                model(x)
        want = model(x).dense_features.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = model(x).dense_features
        for _ in range(2):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


@pytest.mark.parametrize("layer_type", [SelfAttention, CrossAttention])
def test_head_norm_weights_may_be_strided(layer_type):
    """Norm weights that are every second element of something, through the layers that normalise and rotate in one pass."""
    D, H, S = 160, 2, 11
    plain = randomize(layer_type(D, H, 0.0, 0.0, qk_normalization=True, device=DEV, dtype=torch.bfloat16, norm_type="layernorm"))
    strided = copy.deepcopy(plain)
    for norm in (strided.q_norm, strided.k_norm):
        for n in ("weight", "bias"):
            wide = torch.zeros(160, device=DEV, dtype=torch.bfloat16)[::2]
            setattr(norm, n, torch.nn.Parameter(wide.copy_(getattr(norm, n).detach())))
            assert not getattr(norm, n).is_contiguous()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, S, D, generator=g).to(DEV, torch.bfloat16)
    args = (x,) if layer_type is SelfAttention else (x, torch.randn(2, 20, D, generator=g).to(DEV, torch.bfloat16))
    outs = []
    for layer in (strided, plain):
        y = layer(*args)
        y.float().square().mean().backward()
        outs.append([y] + [p.grad for p in layer.parameters()])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
