"""Host side of the relative position bias, the key counts and the per-head normalisation pass: bucket plans against brute
force, and the refusals, which need no GPU."""
import copy
import ctypes
import itertools
import math
import os
import pickle
import re
import subprocess

import pytest
import torch

from vit_amd import KVMemory, RelativeBuckets, ViTConfig, _lib, kernels, ops, qk_norm_rope
from vit_amd.attention import CrossAttention, SelfAttention, attention, attention_q_kv_packed
from vit_amd.transformer import TransformerEncoderLayer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def unsigned(index16):
    return index16.to(torch.int64) & 0xFFFF


@pytest.mark.parametrize("shape,nb", [((1, 1), 1), ((3, 5), 7), ((40, 61), 3), ((200, 300), 65536)])
def test_plan_covers_every_pair_once_in_bucket_order(shape, nb):
    g = torch.Generator().manual_seed(shape[0])
    idx = torch.randint(0, nb, shape, generator=g)
    if nb > 1000:
        idx[0, 0] = nb - 1   # a number that does not fit a signed 16-bit integer
    plan = RelativeBuckets(idx, nb)
    assert plan.shape == shape and plan.num_buckets == nb
    assert torch.equal(unsigned(plan.index16), idx)
    order = plan.order.long()
    assert torch.equal(order.sort().values, torch.arange(idx.numel()))
    flat = idx.reshape(-1)
    assert torch.equal(plan.piece[[0, -1]].long(), torch.tensor([0, idx.numel()])) and plan.piece.numel() == plan.num_pieces + 1
    assert plan.bucket_piece.numel() == nb + 1 and int(plan.bucket_piece[-1]) == plan.num_pieces
    sizes = plan.piece.diff()
    assert int(sizes.min()) >= 1 and int(sizes.max()) <= plan.piece_length
    used = torch.unique(flat).tolist()
    for n in used[:50]:
        a, b = int(plan.bucket_piece[n]), int(plan.bucket_piece[n + 1])
        mine = order[int(plan.piece[a]):int(plan.piece[b])]
        assert torch.equal(mine, (flat == n).nonzero()[:, 0])   # all pairs of the bucket, in rising order
    for n in set(range(min(nb, 50))) - set(used):
        assert plan.bucket_piece[n] == plan.bucket_piece[n + 1]


@pytest.mark.parametrize("dims,prefix,table", [((3, 4), 0, None), ((3, 4), 2, None), ((5,), 1, None), ((2, 3, 2), 0, (4, 3, 3)), ((1, 1), 1, None)])
def test_grid_buckets_are_one_per_offset(dims, prefix, table):
    plan = RelativeBuckets.grid(dims, prefix, table_dims=table)
    idx = unsigned(plan.index16)
    n = math.prod(dims)
    assert plan.shape == (n + prefix,) * 2
    table = table or dims
    assert plan.num_buckets == math.prod(2 * t - 1 for t in table) + (3 if prefix else 0)
    pos = list(itertools.product(*[range(d) for d in dims]))
    seen = {}
    for i, a in enumerate(pos):
        for j, b in enumerate(pos):
            off = tuple(x - y for x, y in zip(a, b))
            assert seen.setdefault(off, int(idx[prefix + i, prefix + j])) == int(idx[prefix + i, prefix + j])
    assert len(set(seen.values())) == len(seen)   # different offsets, different buckets
    if prefix:
        special = {int(idx[0, prefix]), int(idx[prefix, 0]), int(idx[0, 0])}
        assert len(special) == 3 and not special & set(seen.values())
        assert bool((idx[:prefix, prefix:] == idx[0, prefix]).all()) and bool((idx[prefix:, :prefix] == idx[prefix, 0]).all())


def test_log_distance_buckets():
    plan = RelativeBuckets.log_distance(50, 400, num_buckets=32, max_distance=128)
    idx = unsigned(plan.index16)
    assert plan.num_buckets == 32
    for d in range(8):   # the first half of the buckets are single distances
        assert int(idx[49, 49 - d]) == d and (d == 0 or int(idx[0, d]) == 16 + d)
    # 8 further buckets grow by (128 / 8)^(1/8) each: their borders, by hand
    for d in range(8, 400):
        want = min(15, 8 + sum(d >= 8 * 16 ** (k / 8) - 1e-6 for k in range(1, 9)))
        assert int(idx[0, d]) == 16 + want, d
    assert bool((idx[0, 1:].diff() >= 0).all())


def test_plan_refusals():
    with pytest.raises(ValueError, match=r"\[0, 4\)"):
        RelativeBuckets(torch.tensor([[0, 4]]), 4)
    with pytest.raises(ValueError, match=r"\[0, 4\)"):
        RelativeBuckets(torch.tensor([[-1, 3]]), 4)
    with pytest.raises(ValueError, match="empty"):
        RelativeBuckets(torch.zeros((0, 3), dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="num_buckets"):
        RelativeBuckets(torch.zeros((1, 3), dtype=torch.int64), 65537)
    with pytest.raises(ValueError, match="integer"):
        RelativeBuckets(torch.zeros((1, 3)), 4)
    with pytest.raises(ValueError, match="integer"):
        RelativeBuckets(torch.zeros((3,), dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="cover"):
        RelativeBuckets.grid((5, 5), table_dims=(4, 5))
    with pytest.raises(ValueError, match="multiple of 4"):
        RelativeBuckets.log_distance(4, 4, num_buckets=6)


def test_attention_refusals():
    q, k = torch.zeros(2, 3, 4, 8), torch.zeros(2, 5, 4, 8)
    plan = RelativeBuckets(torch.zeros((3, 5), dtype=torch.int64), 2)
    table = torch.zeros(2, 4)
    bad = [
        (dict(q=q[0]), "must be"), (dict(k=torch.zeros(2, 5, 2, 8)), "go with"), (dict(k=torch.zeros(3, 5, 4, 8)), "go with"),
        (dict(v=torch.zeros(2, 6, 4, 8)), "differ"), (dict(bias_table=table), "both"), (dict(buckets=plan), "both"),
        (dict(bias_table=torch.zeros(3, 4), buckets=plan), "bias_table must be"),
        (dict(bias_table=table, buckets=RelativeBuckets(torch.zeros((5, 3), dtype=torch.int64), 2)), "buckets cover"),
        (dict(kv_lengths=torch.zeros(3, dtype=torch.int32)), "kv_lengths"), (dict(kv_lengths=[1, 2]), "kv_lengths"),
        (dict(kv_lengths=torch.zeros(2)), "kv_lengths"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
        (dict(dropout=1.0, training=True), "dropout"), (dict(q=torch.zeros(2, 3, 4, 136), k=torch.zeros(2, 5, 4, 136)), "head_dim"),
    ]
    for change, match in bad:
        kw = dict(q=q, k=k, v=None) | change
        kw["v"] = kw["k"] if kw["v"] is None else kw["v"]
        with pytest.raises(ValueError, match=match):
            attention(**kw)
    with pytest.raises(TypeError, match="float16"):
        attention(q.half(), k.half(), k.half())
    with pytest.raises(TypeError, match="queries"):
        attention(q, k.bfloat16(), k.bfloat16())
    with pytest.raises(RuntimeError, match="no CPU fallback|MI355X"):
        attention(q, k, k)


def test_qk_norm_rope_refusals():
    q, w = torch.zeros(2, 3, 4, 16), torch.ones(16)
    for kw, match in [(dict(q=torch.zeros(2, 3, 4, 12), w=torch.ones(12)), "multiples of 8"), (dict(w=torch.ones(8)), "q_norm_weight"),
                      (dict(k=q), "k_norm_weight"), (dict(rope_q=torch.zeros(2, 4, 16)), "rope_q"),
                      (dict(rope_q=torch.zeros(2, 3, 1, 2, 16)), "rope_q"), (dict(eps=-1.0), "eps"),
                      (dict(q_norm_bias=torch.zeros(16, dtype=torch.bfloat16)), "q_norm_bias")]:
        kw = dict(kw)
        with pytest.raises(ValueError, match=match):
            qk_norm_rope(kw.pop("q", q), kw.pop("k", None), kw.pop("w", w), **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback|MI355X"):
        qk_norm_rope(q, None, w)


def test_layer_refusals():
    x = torch.zeros(1, 5, 32)
    plan = RelativeBuckets(torch.zeros((5, 5), dtype=torch.int64), 3)
    with pytest.raises(ValueError, match="relative position bias"):
        SelfAttention(32, 2, relative_buckets=3)(x)
    with pytest.raises(ValueError, match="relative position bias"):
        SelfAttention(32, 2)(x, buckets=plan)
    with pytest.raises(ValueError, match="sequence of 4"):
        SelfAttention(32, 2, relative_buckets=3)(x[:, :4], buckets=plan)
    with pytest.raises(NotImplementedError, match="relative"):
        SelfAttention(32, 2, relative_buckets=3).forward_weights(x)
    layer = CrossAttention(32, 2).eval()
    memory = KVMemory(torch.zeros(1, 7, 2, 2, 16), None)
    with torch.no_grad(), pytest.raises(ValueError, match="project_kv"):
        layer(x, memory, kv_lengths=torch.tensor([1]))
    with torch.no_grad(), pytest.raises(ValueError, match="go with"):
        layer(x, KVMemory(torch.zeros(2, 7, 2, 2, 16), None))
    with pytest.raises(RuntimeError, match="inference"):
        layer(x, memory)
    with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
        layer.train()(x, memory)
    with pytest.raises(ValueError, match="kv_lengths"):
        layer(x, x, kv_lengths=torch.tensor([1, 2]))


def test_relative_vit_has_a_table_per_block_and_refuses_masks():
    cfg = ViTConfig(in_channels=3, patch_size=(8, 8), img_size=(32, 24), depth=2, hidden_size=64, ffn_hidden_size=128,
                    num_attention_heads=2, num_register_tokens=2, pos_enc="relative", dtype=torch.float32)
    model = cfg.instantiate()
    names = [n for n in model.state_dict() if "relative" in n]
    assert names == [f"blocks.{i}.self_attention.relative_bias" for i in range(2)]
    assert tuple(model.state_dict()[names[0]].shape) == (7 * 5 + 3, 2)
    assert ViTConfig.from_yaml(cfg.to_yaml()) == cfg
    assert model.prepare_buckets((4, 3)).shape == (14, 14)
    assert model.prepare_buckets((2, 3)).num_buckets == 38 and model.prepare_buckets((4, 3)) is model.prepare_buckets((4, 3))
    with pytest.raises(ValueError, match="cover"):
        model.prepare_buckets((5, 3))
    with pytest.raises(NotImplementedError, match="masks"):
        model(torch.zeros(1, 3, 32, 24), mask=torch.ones(1, 12, dtype=torch.bool))
    assert not [n for n in ViTConfig(**{**cfg.__dict__, "pos_enc": "rope"}).instantiate().state_dict() if "relative" in n]


@pytest.mark.parametrize("cname", ["VitkQkSection", "VitkQkNormRope", "VitkAttnVar"])
def test_descriptor_layout_matches_the_header(cname):
    header = open(os.path.join(ROOT, "include", "vitk.h")).read()
    body = header[header.index(f"typedef struct {cname} {{"):header.index(f"}} {cname};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for stmt in body.split("{", 1)[1].split(";"):
        if stmt.strip():
            names += [re.sub(r"\[\d+\]|[*\s]", "", piece.split()[-1]) for piece in stmt.split(",")]
    assert names == [f[0] for f in getattr(_lib, cname)._fields_]


def test_entry_points_refuse_bad_descriptors():
    """Errors of the C entry points come back as a code and a text; nothing is launched for them."""
    lib = _lib.load()

    def err(rc):
        return lib.vitk_last_error().decode() if rc else ""

    a = _lib.VitkAttnVar()
    a.B, a.H, a.Lq, a.Lk, a.Dh, a.scale = 1, 1, 1, 1, 129, 1.0
    assert "bad shape" in err(lib.vitk_attn_var_fwd(ctypes.byref(a), None)) and "null" in err(lib.vitk_attn_var_fwd(None, None))
    a.Dh = 64
    assert "null pointer" in err(lib.vitk_attn_var_fwd(ctypes.byref(a), None))
    a.Lq = 1 << 22
    assert "at most" in err(lib.vitk_attn_var_bwd(ctypes.byref(a), None))
    a.Lq, a.scale = 1, 0.0
    assert "scale" in err(lib.vitk_attn_var_fwd(ctypes.byref(a), None))
    a.scale, a.drop_p = 1.0, 1.0
    assert "dropout" in err(lib.vitk_attn_var_fwd(ctypes.byref(a), None))
    a.drop_p, a.dtype = 0.0, 7
    assert "dtype" in err(lib.vitk_attn_var_fwd(ctypes.byref(a), None))
    n = _lib.VitkQkNormRope()
    n.B, n.Dh = 1, 20
    assert "multiple of 8" in err(lib.vitk_qk_norm_rope_fwd(ctypes.byref(n), None)) and "null" in err(lib.vitk_qk_norm_rope_bwd(None, None))
    n.Dh = 16
    assert "null pointer" in err(lib.vitk_qk_norm_rope_fwd(ctypes.byref(n), None))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("B,Lq,Lk", [(0, 5, 500), (3, 0, 500), (3, 5, 0), (0, 0, 0), (0, 500, 500), (1, 1, 1)])
def test_workspace_of_empty_problems(B, Lq, Lk, dtype):
    """Sizes of zero pass every rule that shares an axis out: no division by the count of nothing."""
    lib = _lib.load()
    a = _lib.VitkAttnVar()
    a.B, a.H, a.Lq, a.Lk, a.Dh, a.scale, a.dtype = B, 2, Lq, Lk, 64, 0.125, dtype
    fake = 1 << 12   # never followed: these calls only count bytes
    a.q = a.k = a.v = a.o = a.stat = a.dout = a.dq = a.dk = a.dv = fake
    for i in range(24):
        a.st[i] = 128
    for table in (None, fake):
        a.bias_table = a.bias_index = a.dbias_table = a.order = a.piece = a.bucket_piece = table
        a.num_buckets = a.num_pieces = 3
        for bwd in (0, 1):
            n = lib.vitk_attn_var_workspace_bytes(ctypes.byref(a), bwd)
            assert n == 0 or bwd or B * Lq * Lk > 0


def test_plans_of_captured_graphs_are_never_dropped(monkeypatch):
    """A model keeps its last eight plans, and every plan that a graph was captured with: replays read its memory."""
    model = ViTConfig(in_channels=3, patch_size=(8, 8), img_size=(32, 32), depth=1, hidden_size=64, ffn_hidden_size=128,
                      num_attention_heads=2, pos_enc="relative", dtype=torch.float32).instantiate()
    capturing = [True]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    first = model.prepare_buckets((1, 2))
    capturing[0] = False
    plans = {g: model.prepare_buckets(g) for g in [(a, b) for a in (1, 2, 3) for b in (1, 2, 3, 4)] if g != (1, 2)}
    assert model.prepare_buckets((1, 2)) is first
    assert model.prepare_buckets((3, 4)) is plans[(3, 4)] and model.prepare_buckets((1, 1)) is not plans[(1, 1)]
    assert len(model._bucket_plans) <= 9


SHARES = r"""
#include "attn_share.h"
#include <cstdio>
#include <initializer_list>
static int fail(int n, int tile, int shares, int y) { std::printf("keys %d tile %d share %d of %d\n", n, tile, y, shares); return 1; }
static int look(int n, int tile, int shares) {
  const int tiles = (n + tile - 1) / tile;
  int at = 0, least = tiles, most = 0;
  for (int y = 0; y < shares; y++) {
    const KeyShare s = key_share(n, tile, shares, y);
    // the tiles follow each other, their keys are covered, and no descriptor reaches behind the last key
    if (s.t0 != at || s.t1 < s.t0 || s.end > n || s.end < 0) return fail(n, tile, shares, y);
    if (s.end != (s.t1 * tile < n ? s.t1 * tile : n)) return fail(n, tile, shares, y);
    if (s.t1 > s.t0 && (s.end <= (s.t1 - 1) * tile)) return fail(n, tile, shares, y);   // its last tile has a key
    at = s.t1;
    least = s.t1 - s.t0 < least ? s.t1 - s.t0 : least;
    most = s.t1 - s.t0 > most ? s.t1 - s.t0 : most;
  }
  return at != tiles || most - least > 1 ? fail(n, tile, shares, -1) : 0;
}
int main() {
  const int tile[] = {32, 64}, large[] = {65537, 999999, (1 << 24) - 1};
  for (int t : tile)
    for (int shares = 1; shares <= 64; shares++) {
      for (int tiles = 0; tiles <= 700; tiles++)
        for (int n : {tiles * t - t + 1, tiles * t - 1, tiles * t})
          if (n >= 0 && look(n, t, shares)) return 1;
      for (int n : large)
        if (look(n, t, shares)) return 1;
    }
  std::puts("covered");
}
"""


def test_key_shares_cover_every_key_once_and_nothing_behind_the_last(tmp_path):
    """The arithmetic by which workgroups share a sample's keys, compiled for the host from the kernels' own header: all tile
    counts and shares; shares without tiles are among them (more shares than tiles)."""
    src = tmp_path / "shares.cc"
    src.write_text(SHARES)
    out = str(tmp_path / "shares")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "vit_amd", "csrc"), str(src), "-o", out], check=True)
    done = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0 and done.stdout == "covered\n", done.stdout


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operands_start_on_16_byte_boundaries(dtype):
    """Contiguous or not, what starts or steps off a boundary is copied; everything else is passed on as it is, axes of one
    element with any stride among it."""
    flat = torch.arange(1 + 2 * 5 * 3 * 64, dtype=torch.float32).to(dtype)
    for off in range(9):
        t = flat[off:off + 2 * 5 * 2 * 64].view(2, 5, 2, 64)
        got = kernels.attn_operand(t)
        assert got.data_ptr() % 16 == 0 and torch.equal(got, t)
        assert (got is t) == (off * t.element_size() % 16 == 0)
    wide = torch.zeros(2, 5, 3, 68, dtype=dtype)[..., :64]
    got = kernels.attn_operand(wide)
    assert (got is wide) == (dtype == torch.float32) and all(s * got.element_size() % 16 == 0 for s in got.stride()[:3])
    one = flat[:64].as_strided((1, 1, 1, 64), (3, 5, 7, 1))
    assert kernels.attn_operand(one) is one
    odd = flat[1:1 + 2 * 5 * 3 * 20].view(2, 5, 3, 20)[..., :12 if dtype == torch.bfloat16 else 10]
    assert kernels.attn_operand(odd) is odd   # head sizes that no 16-byte access fits
    leaf = flat[1:129].view(1, 2, 1, 64).clone().requires_grad_(True)
    shifted = torch.cat([leaf.new_zeros(1), leaf.reshape(-1)])[1:].view(1, 2, 1, 64)
    kernels.attn_operand(shifted).square().sum().backward()
    assert torch.equal(leaf.grad, 2 * leaf.detach())


def test_rotation_tables_start_on_16_byte_boundaries():
    for shape, keep in (((2, 5, 16), None), ((2, 3, 1, 5, 16), None), ((2, 3, 1, 5, 16), torch.tensor([2, 0]))):
        n = math.prod(shape)
        rope = torch.arange(n + 1.0)[1:].view(shape)
        assert rope.is_contiguous() and rope.data_ptr() % 16
        table, _ = ops._rope_table(rope, keep, 3, 3 if keep is None else 2, torch.float32)
        want = rope if len(shape) == 3 else rope[:, :, 0] if keep is None else rope[:, keep, 0]
        assert table.data_ptr() % 16 == 0 and torch.equal(table, want)
    aligned = torch.zeros(2, 5, 16)
    assert ops._rope_table(aligned, None, 3, 3, torch.float32)[0].data_ptr() == aligned.data_ptr()


@pytest.mark.parametrize("shape", [(2, 3, 16), (2, 2, 1, 3, 16)])
def test_rotation_tables_that_ask_for_a_gradient_are_refused(shape):
    """They would get none; where no gradients are taken, and detached, they pass (as far as the missing GPU)."""
    q, w, rope = torch.zeros(2, 3, 4, 16), torch.ones(16), torch.zeros(shape, requires_grad=True)
    for kw in (dict(rope_q=rope), dict(k=q, k_norm_weight=w, rope_k=rope)):
        with pytest.raises(ValueError, match="constant table"):
            qk_norm_rope(q, kw.pop("k", None), w, **kw)
    for context, table in ((torch.no_grad(), rope), (torch.enable_grad(), rope.detach())):
        with context, pytest.raises(RuntimeError, match="no CPU fallback|MI355X"):
            qk_norm_rope(q, None, w, rope_q=table)


def test_zero_padding_refusals():
    lib = _lib.load()
    for args, match in (((None, None, None, 1, 1, 3), "bad shape"), ((None, None, None, -1, 1, 4), "bad shape"), ((None, None, None, 1, 1, 4), "null"),
                        ((4097, 4096, 4096, 1, 1, 4), "aligned")):
        assert lib.vitk_zero_padding(*args, None) != 0 and match in lib.vitk_last_error().decode()
    assert lib.vitk_zero_padding(None, None, None, 0, 5, 4, None) == 0 and lib.vitk_zero_padding(None, None, None, 5, 0, 4, None) == 0


def test_head_norms_of_padded_rows_need_an_eps():
    """A padded row is cleared before its gradient is formed; without an eps the norm of zeros is no number."""
    q, kv, w = torch.zeros(2, 3, 32), torch.zeros(2, 4, 32), torch.zeros(32, 32, requires_grad=True)
    ones = torch.ones(16)
    args = (w, None, torch.zeros(64, 32), None, torch.ones(32), None, False, 16, w, None, None, 1e-5, ones, None, ones, None, False)
    lens = torch.tensor([4, 1])
    for eps, wkv_grad, error in ((0.0, True, ValueError), (1e-5, True, RuntimeError), (0.0, False, RuntimeError)):
        a = list(args)
        a[2] = torch.zeros(64, 32, requires_grad=wkv_grad)
        with pytest.raises(error, match="qk_eps" if error is ValueError else "no CPU fallback|MI355X"):
            attention_q_kv_packed(q, kv, *a, eps, True, 0.0, 0.0, True, kv_lengths=lens)


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("pos_enc", ["none", "relative"])
def test_blocks_without_a_relative_bias_are_called_as_ever(pos_enc, ckpt):
    """A model whose blocks override forward(x, rope) runs; with a relative bias they get its plan."""
    seen = []

    class Block(TransformerEncoderLayer):
        def forward(self, x, rope=None):
            seen.append(None)
            return x + 1

    class BiasBlock(TransformerEncoderLayer):
        def forward(self, x, rope=None, buckets=None):
            seen.append(buckets)
            return x + 1

    class Stem(torch.nn.Module):
        def tokenized_size(self, size):
            return tuple(s // 8 for s in size)

        def forward(self, x, prefix=None):
            return torch.zeros(1, 12, 64, requires_grad=True)

    model = ViTConfig(in_channels=3, patch_size=(8, 8), img_size=(32, 24), depth=2, hidden_size=64, ffn_hidden_size=128,
                      num_attention_heads=2, pos_enc=pos_enc, dtype=torch.float32, activation_checkpointing=ckpt).instantiate().train()
    model.stem = Stem()
    model.blocks = torch.nn.ModuleList([(BiasBlock if pos_enc == "relative" else Block)(64, 128, 2) for _ in range(2)])
    out = model(torch.zeros(1, 3, 32, 24), output_norm=False)
    assert bool((out.dense_features == 2).all())
    assert [s if s is None else s.shape for s in seen] == [None if pos_enc == "none" else (12, 12)] * 2


def test_plans_are_made_under_any_default_device():
    """The index decides where a plan lives, not torch's default device (meta stands for a GPU here)."""
    index = torch.randint(0, 9, (20, 30), generator=torch.Generator().manual_seed(1))
    made = lambda: (RelativeBuckets(index, 9), RelativeBuckets.grid((3, 4), 2, device="cpu"), RelativeBuckets.log_distance(20, 30, device="cpu"))
    want = made()
    with torch.device("meta"):
        got = made()
    for a, b in zip(got, want):
        for n in ("index16", "order", "piece", "bucket_piece"):
            assert torch.equal(getattr(a, n), getattr(b, n)), n


def test_copies_and_saved_models_carry_no_plans():
    model = ViTConfig(in_channels=3, patch_size=(8, 8), img_size=(256, 256), depth=1, hidden_size=64, ffn_hidden_size=128,
                      num_attention_heads=2, pos_enc="relative", dtype=torch.float32).instantiate()
    size = lambda: len(pickle.dumps(model))
    before = size()
    plan = model.prepare_buckets((32, 32))
    assert size() - before < 4096 and model.prepare_buckets((32, 32)) is plan
    for other in (copy.deepcopy(model), pickle.loads(pickle.dumps(model))):
        assert other._bucket_plans == {} and other._captured_plans == set() and other.prepare_buckets((32, 32)) is not plan
        assert all(torch.equal(a, b) for a, b in zip(other.state_dict().values(), model.state_dict().values()))
    assert model.prepare_buckets((32, 32)) is plan
