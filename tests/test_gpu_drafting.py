"""The drafting operators together, as a decoder would use them.

  * The depth stack over a tree of drafts: the model's own weights (as they are, or in
    4 bits), its bias by distance, tree_attention over caches that cache_commit filled.
    Every node's logits are those of the full pass over its path, the oracle's and, in the
    weights' own type, depth_forward_full's.  Tolerances are those of depth_forward_full
    itself, norm-wise: fp32 1e-4, bf16 2e-2, fp16 5e-3; between two results that each may
    be off by that, twice as much.
  * Steps of a decoder held to a budget: 4-bit projections, attention, commit with
    weights, eviction; each step against 64 bits from the state that it began with, and
    captured graphs, two at once, against the same steps run eagerly.
"""

from __future__ import annotations

import dataclasses
import math

import numpy as np
import pytest
import torch

import mrt_df
import synth_bundle
from oracle import depthformer_oracle as DO
from oracle import drafting_oracle as O
from test_gpu_cache_ops import check_evict
from test_gpu_tree_attention import DEV, DT

pytestmark = pytest.mark.gpu
TOL = {"fp32": 1e-4, "bf16": 2e-2, "fp16": 5e-3}


def rel(a, b):
    a, b = (np.asarray(x, dtype=np.float64) for x in (a, b))
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


class DepthStack:
    """The depth layers over caches of the caller's own; `q4`: products with 4-bit weights."""

    def __init__(self, w, cfg, dtype, q4, bias, rows, room):
        self.cfg, self.dt, self.bias = cfg, DT[dtype], bias
        names = [n for n in w if n.startswith("depth_layers.") or n in ("decoder_norm.weight", "lm_head.weight")]
        self.w = {n: torch.tensor(np.asarray(w[n], dtype=np.float32)).to(DEV, self.dt) for n in names}
        self.codes = {n: mrt_df.q4_quantize(x, 64) for n, x in self.w.items() if q4 and x.dim() == 2}
        shape = (rows, cfg.num_heads, room, cfg.d_kv)
        self.kv = [(torch.zeros(shape, dtype=self.dt, device=DEV), torch.zeros(shape, dtype=self.dt, device=DEV))
                   for _ in range(cfg.num_depth_layers)]
        self.length = torch.zeros(rows, dtype=torch.int32, device=DEV)

    def lin(self, x, name):
        if name + ".weight" in self.codes:
            rows = x.reshape(-1, x.shape[-1])
            got = torch.cat([mrt_df.q4_matmul(rows[i:i + 64], *self.codes[name + ".weight"]) for i in range(0, len(rows), 64)])
            return got.view(*x.shape[:-1], -1)
        return (x.float() @ self.w[name + ".weight"].float().T).to(self.dt)

    def norm(self, x, name):
        f = x.float()
        return (f * (f.square().mean(-1, keepdim=True) + 1e-6).rsqrt()).to(self.dt) * self.w[name + ".weight"]

    def forward(self, x, parents):
        """Logits of every node of x (rows, nodes, d_model); its K/V stay in self.fresh."""
        cfg, self.fresh = self.cfg, []
        parents = torch.tensor(parents, dtype=torch.int32, device=DEV)
        heads = lambda y: y.view(*y.shape[:2], cfg.num_heads, cfg.d_kv)  # noqa: E731
        for i, kv in enumerate(self.kv):
            p = f"depth_layers.{i}."
            y = self.norm(x, p + "pre_self_attn_norm")
            q, k, v = (heads(self.lin(y, p + f"self_attn.{n}_proj")) for n in "qkv")
            self.fresh.append((k, v))
            o, _ = mrt_df.tree_attention(q, k, v, mrt_df.KVCache(*kv, self.length), parents, bias=self.bias)
            x = x + self.lin(o.flatten(2), p + "self_attn.o_proj")
            y = self.norm(x, p + "pre_ffn_norm")
            y = torch.nn.functional.gelu(self.lin(y, p + "ffn.wi_0").float(), approximate="tanh").to(self.dt) \
                * self.lin(y, p + "ffn.wi_1")
            x = x + self.lin(y, p + "ffn.wo")
        return self.lin(self.norm(x, "decoder_norm"), "lm_head").float().cpu().numpy()

    def commit(self, path):
        rows = self.length.shape[0]
        took = torch.tensor([path] * rows, dtype=torch.int32, device=DEV)
        length = torch.empty_like(self.length)
        for kv, (k, v) in zip(self.kv, self.fresh):
            mrt_df.cache_commit(mrt_df.KVCache(*kv, self.length), k, v, took, length)
        self.length = length


@pytest.mark.parametrize("q4", [False, True], ids=["weights", "q4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_depth_stack_over_a_tree(dtype, q4):
    cfg = mrt_df.Config.tiny()
    w = synth_bundle.make_weights(cfg, seed=21, norm_jitter=0.1)
    m = mrt_df.Depthformer(w, cfg, dtype=dtype)
    bias = m.precompute_biases("depth", 16)[15].flip(1).float().contiguous()  # (heads, distance)
    stack = DepthStack(w, cfg, dtype, q4, bias, rows=2, room=16)
    ow = dict(w)
    for n, c in stack.codes.items():
        ow[n] = O.q4_weights(*(x.cpu() for x in c)).float().numpy()
    # dequantized weights are not values of a 16-bit type: the oracle keeps them in fp32
    om = DO.OracleDepthformer(ow, DO.DepthformerConfig(**dataclasses.asdict(cfg)), mode="fp32" if q4 else dtype)
    rng = np.random.default_rng(5)
    embs = DO.Precision(dtype).r(rng.standard_normal((2, 5 + 11, cfg.d_model)).astype(np.float32))
    x = torch.tensor(embs).to(DEV, DT[dtype])
    chain, tree = list(range(-1, 4)), [-1, 0, 0, 2, -1, 4, 3, 6, 7, 5, 8]
    logits = np.concatenate([stack.forward(x[:, :5], chain), np.zeros((2, 11, cfg.vocab_size))], 1)
    stack.commit([0, 1, 2, 3, 4])
    logits[:, 5:] = stack.forward(x[:, 5:], tree)
    st = m.new_state(max_frames=2)
    for t, path in enumerate(O.chains(tree)):
        at = [0, 1, 2, 3, 4] + [5 + u for u in path]
        want = om.depth_forward_full(embs[:, at])
        for j in (0, 4, len(at) - 1):
            assert rel(logits[:, at[j]], want[:, j]) <= TOL[dtype], (t, j)
        if not q4:
            full = st.depth_forward_full(x[:, at].contiguous()).cpu().numpy()
            assert rel(logits[:, at[-1]], full[:, -1]) <= 2 * TOL[dtype], t
    # a committed path is what the next drafts see
    stack.commit([0, 2, 3])
    assert stack.length.tolist() == [8, 8]
    more = stack.forward(x[:, :1], [-1])
    want = om.depth_forward_full(np.concatenate([embs[:, [0, 1, 2, 3, 4, 5, 7, 8]], embs[:, :1]], 1))
    assert rel(more[:, 0], want[:, -1]) <= TOL[dtype]
    st.close()
    m.close()


class Decoder:
    """One attention layer held to `budget` entries; a step is a fixed sequence of calls on
    fixed buffers, so that it can be captured."""

    ROWS, HEADS, KV, D, NODES = 3, 8, 2, 64, 9
    MODEL, CAP, BUDGET, RECENT, SINKS = 256, 2600, 2400, 100, 4

    def __init__(self, seed, dtype):
        g = torch.Generator().manual_seed(seed)
        dt, d, kv = DT[dtype], self.D, self.KV
        wide = (self.HEADS + 2 * kv) * d
        self.codes = mrt_df.q4_quantize((torch.randn((wide, self.MODEL), generator=g) / 16).to(DEV, dt), 32)
        self.back = mrt_df.q4_quantize((torch.randn((self.MODEL, self.HEADS * d), generator=g) / 22).to(DEV, dt), 64)
        slots = (self.ROWS, kv, self.CAP)
        self.k, self.v = (torch.randn((*slots, d), generator=g).to(DEV, dt) for _ in range(2))
        self.length = torch.tensor([2397, 0, 1200], dtype=torch.int32, device=DEV)
        self.next = self.length.clone()
        self.pos = torch.arange(self.CAP, dtype=torch.int32, device=DEV).expand(slots).contiguous()
        self.score = torch.rand(slots, generator=g).to(DEV)
        self.length2, self.next2 = torch.empty_like(self.length), torch.empty_like(self.length)
        self.x = torch.randn((self.ROWS, self.NODES, self.MODEL), generator=g).to(DEV, dt)
        self.bias = (torch.randn((self.HEADS, 128), generator=g) / 4).to(DEV)
        self.parents = torch.tensor([-1, 0, 1, 1, 0, -1, 5, 3, 7], dtype=torch.int32, device=DEV)
        self.accepted = torch.tensor([[0, 1, 3, 7], [5, 6, -1, -1], [-1, -1, -1, -1]], dtype=torch.int32, device=DEV)
        self.kw = dict(scale=1 / math.sqrt(d), bias=self.bias)

    def step(self):
        h, kv, d = self.HEADS, self.KV, self.D
        y = mrt_df.q4_matmul(self.x.view(-1, self.MODEL), *self.codes).view(self.ROWS, self.NODES, -1)
        self.q = y[..., :h * d].unflatten(-1, (h, d))
        self.kn, self.vn = (y[..., (h + z * kv) * d:(h + (z + 1) * kv) * d].unflatten(-1, (kv, d)) for z in range(2))
        cache = mrt_df.KVCache(self.k, self.v, self.length, self.pos, self.next, self.score)
        out, lse = mrt_df.tree_attention(self.q, self.kn, self.vn, cache, self.parents, **self.kw)
        mrt_df.cache_commit(cache, self.kn, self.vn, self.accepted, self.length2, self.next2, self.q, lse, self.score, **self.kw)
        grown = mrt_df.KVCache(self.k, self.v, self.length2, self.pos, self.next2, self.score)
        mrt_df.cache_evict(grown, self.BUDGET, self.length, self.score, self.pos, recent=self.RECENT, sinks=self.SINKS)
        self.next.copy_(self.next2)
        self.x.copy_(mrt_df.q4_matmul(out.view(-1, h * d), *self.back).view_as(self.x).tanh())
        self.out, self.lse = out, lse

    def state(self):
        torch.cuda.synchronize()
        return {n: getattr(self, n).cpu().clone() for n in ("k", "v", "length", "next", "pos", "score", "x")}


@pytest.mark.parametrize("dtype", ["bf16", "fp32", "fp16"])
def test_decoder_steps_against_64_bits(dtype):
    """Whole numbers and moved rows equal.  Scores: the accepted tokens' weights, each off by
    the logits' rounding: sums of 64 products and five more roundings of values up to
    `big`, and the logarithm of the sum; 17 terms of a sum.  The outputs' own accuracy is
    tested with the operators; here, half a step of the type beside the weights' error."""
    dec = Decoder(3, dtype)
    for step in range(4):
        was = dec.state()
        dec.step()
        now = dec.state()
        q, kn, vn, lse, out = (x.cpu() for x in (dec.q, dec.kn, dec.vn, dec.lse, dec.out))
        kw = dict(scale=dec.kw["scale"], bias=dec.bias.cpu(), pos=was["pos"], next_pos=was["next"])
        want, lse64 = O.tree_attention(q, kn, vn, was["k"], was["v"], was["length"], dec.parents.cpu(), **kw)
        norm = lambda *xs: max(float(x.double().norm(dim=-1).max()) for x in xs)  # noqa: E731
        big = kw["scale"] * norm(q) * norm(was["k"], kn) + float(dec.bias.abs().max()) + float(lse64.abs().max())
        delta = 2 * (64 + 8) * 2.0 ** -24 * big + 2.0 ** -16 + 2420 * 2.0 ** -24
        top = max(float(was["v"].double().abs().max()), float(vn.double().abs().max()))
        assert ((out.double() - want).abs() <= torch.finfo(DT[dtype]).eps / 2 * want.abs() + 2 * delta * top).all()
        grown = O.cache_commit(was["k"], was["v"], was["length"], kn, vn, dec.accepted.cpu(), q=q, lse=lse,
                               score=was["score"], score_out=was["score"], **kw)
        # what the commit left, which is what the eviction went by: the same call once more
        again = Decoder(3, dtype)
        for n in was:
            getattr(again, n).copy_(was[n].to(DEV))
        cache = mrt_df.KVCache(again.k, again.v, again.length, again.pos, again.next, again.score)
        mrt_df.cache_commit(cache, dec.kn, dec.vn, dec.accepted, again.length2, again.next2, dec.q, dec.lse, again.score,
                            **again.kw)
        torch.cuda.synchronize()
        mid = dict(k=again.k.cpu(), v=again.v.cpu(), length=again.length2.cpu(), pos=again.pos.cpu(),
                   next_pos=again.next2.cpu(), score=again.score.cpu())
        for n in ("k", "v", "length", "pos", "next_pos"):
            assert torch.equal(mid[n], grown[n]), n
        for b, n in enumerate(grown["length"].tolist()):
            err = (mid["score"][b, :, :n].double() - grown["score"][b, :, :n]).abs()
            assert (err <= (delta + 17 * 2.0 ** -24) * grown["score"][b, :, :n]).all()
        check_evict(mid, dict(now, next_pos=None), dec.BUDGET, dec.RECENT, dec.SINKS, untouched=False)
        assert torch.equal(now["next"], grown["next_pos"])
        assert now["length"].max() <= dec.BUDGET
    assert now["length"].tolist() == [2400, 8, 1200] and now["next"].tolist() == [2413, 8, 1200]


def test_captured_decoders_replay_at_once():
    """Two graphs with workspaces of their own, replayed side by side, with eager work
    between the replays: bit for bit what the steps give when run one by one."""
    seeds, steps = (3, 4), 4
    want = []
    for seed in seeds:
        dec = Decoder(seed, "bf16")
        states = []
        for _ in range(steps):
            dec.step()
            states.append(dec.state())
        want.append(states)
    decs, graphs, streams = [Decoder(s, "bf16") for s in seeds], [], [torch.cuda.Stream() for _ in seeds]
    for dec, stream in zip(decs, streams):
        first = dec.state()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            dec.step()  # warm, then back to the start
            for n, x in first.items():
                getattr(dec, n).copy_(x.to(DEV))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            dec.step()
        graphs.append(graph)
        torch.cuda.synchronize()
    other = Decoder(9, "fp16")
    for i in range(steps):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        other.step()
        for dec, states in zip(decs, want):
            got = dec.state()
            for n, x in states[i].items():
                assert torch.equal(got[n], x), (i, n)
