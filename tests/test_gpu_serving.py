"""The operators of a server's step together, as a server would use them.

  * The model's depth stack with its caches in pages: entries written and attended chunk by
    chunk and token by token, each logit that of the full pass.  Tolerances are those of
    depth_forward_full itself, norm-wise: fp32 1e-4, bf16 2e-2, fp16 5e-3.
  * Steps of a server that drafts: 8-bit products, pages of codes, attention, verification,
    batches padded.  Every call of a step against 64 bits from what it was given, and
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
from oracle import serving_oracle as O
from test_gpu_drafting import TOL, DepthStack, rel
from test_gpu_i8 import check as check_product
from test_gpu_paged import DEV, DT, check as check_attention, same

pytestmark = pytest.mark.gpu


class PagedStack(DepthStack):
    """The depth layers over pages of 16 entries, which the sequences take in turns."""

    def __init__(self, w, cfg, dtype, bias, rows, room):
        super().__init__(w, cfg, dtype, False, bias, rows, room)
        table = torch.arange(rows * room // 16, dtype=torch.int32, device=DEV).view(-1, rows).T.contiguous()
        pool = (table.numel(), cfg.num_heads, 16, cfg.d_kv)
        self.pages = [(torch.zeros(pool, dtype=self.dt, device=DEV), torch.zeros(pool, dtype=self.dt, device=DEV), table)
                      for _ in range(cfg.num_depth_layers)]

    def forward(self, x, fresh=None):
        cfg = self.cfg
        heads = lambda y: y.view(*y.shape[:2], cfg.num_heads, cfg.d_kv)  # noqa: E731
        grown = torch.empty_like(self.length)
        for i, (k_pool, v_pool, table) in enumerate(self.pages):
            p = f"depth_layers.{i}."
            y = self.norm(x, p + "pre_self_attn_norm")
            q, k, v = (heads(self.lin(y, p + f"self_attn.{n}_proj")) for n in "qkv")
            cache = mrt_df.PagedCache(k_pool, v_pool, table, self.length)
            mrt_df.paged_write(cache, k, v, fresh=fresh, length_out=grown)
            o, _ = mrt_df.paged_attention(q, cache, fresh=fresh, bias=self.bias)
            x = x + self.lin(o.flatten(2), p + "self_attn.o_proj")
            y = self.norm(x, p + "pre_ffn_norm")
            y = torch.nn.functional.gelu(self.lin(y, p + "ffn.wi_0").float(), approximate="tanh").to(self.dt) \
                * self.lin(y, p + "ffn.wi_1")
            x = x + self.lin(y, p + "ffn.wo")
        self.length = grown
        return self.lin(self.norm(x, "decoder_norm"), "lm_head").float().cpu().numpy()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_depth_stack_over_pages(dtype):
    cfg = mrt_df.Config.tiny()
    w = synth_bundle.make_weights(cfg, seed=21, norm_jitter=0.1)
    m = mrt_df.Depthformer(w, cfg, dtype=dtype)
    bias = m.precompute_biases("depth", 16)[15].flip(1).float().contiguous()  # (heads, distance)
    m.close()
    stack = PagedStack(w, cfg, dtype, bias, rows=3, room=32)
    om = DO.OracleDepthformer(w, DO.DepthformerConfig(**dataclasses.asdict(cfg)), mode=dtype)
    embs = DO.Precision(dtype).r(np.random.default_rng(5).standard_normal((3, 16, cfg.d_model)).astype(np.float32))
    x = torch.tensor(embs).to(DEV, DT[dtype])
    want, at = om.depth_forward_full(embs), [0, 0, 0]
    for fresh in ([7, 1, 0], [1, 1, 1], [1, 1, 1], [4, 7, 2], [0, 3, 7], [3, 1, 4]):
        n = max(fresh)
        step = torch.stack([torch.nn.functional.pad(x[b, at[b]:at[b] + fresh[b]], (0, 0, 0, n - fresh[b])) for b in range(3)])
        got = stack.forward(step, None if min(fresh) == n else torch.tensor(fresh, dtype=torch.int32, device=DEV))
        for b in range(3):
            for t in range(fresh[b]):
                assert rel(got[b, t], want[b, at[b] + t]) <= TOL[dtype], (fresh, b, t)
            at[b] += fresh[b]
        assert stack.length.tolist() == at


class Server:
    """One layer and the head of a server that drafts NODES tokens a step; a step is a fixed
    sequence of calls on fixed buffers, so that it can be captured."""

    ROWS, HEADS, KV, D, NODES, MODEL, VOCAB, PAGE, ROW_PAGES = 3, 8, 2, 64, 4, 256, 41000, 64, 50

    def __init__(self, seed, dtype, store):
        g = torch.Generator().manual_seed(seed)
        self.dt, d, kv, slots = DT[dtype], self.D, self.KV, self.NODES + 1
        wide = (self.HEADS + 2 * kv) * d
        weight = lambda n, k: mrt_df.i8_quantize((torch.randn((n, k), generator=g) / math.sqrt(k)).to(DEV, self.dt))  # noqa: E731
        self.w_in, self.w_back, self.w_head = weight(wide, self.MODEL), weight(self.MODEL, self.HEADS * d), weight(self.VOCAB, self.MODEL)
        self.emb = torch.randn((self.VOCAB, self.MODEL), generator=g).to(DEV, self.dt)
        pages = self.ROWS * self.ROW_PAGES
        pool = (pages, kv, self.PAGE, d)
        values = [torch.randn(pool, generator=g).to(DEV, self.dt) for _ in range(2)]
        self.k_scale = self.v_scale = None
        if store == "i8":
            (self.k, self.k_scale), (self.v, self.v_scale) = (
                (c.view(pool), s.view(pool[:3])) for c, s in (mrt_df.i8_quantize(x.view(-1, d)) for x in values))
        else:
            self.k, self.v = values
        self.table = torch.randperm(pages, generator=g).view(self.ROWS, -1).to(DEV, torch.int32)
        self.length = torch.tensor([2900, 0, 1500], dtype=torch.int32, device=DEV)
        self.grown = torch.empty_like(self.length)
        self.fresh = torch.tensor([slots, 3, 1], dtype=torch.int32, device=DEV)
        self.slot = torch.arange(self.NODES, device=DEV)
        self.token = torch.tensor([5, 6, 7], dtype=torch.int32, device=DEV)
        self.bias = (torch.randn((self.HEADS, 128), generator=g) / 4).to(DEV)
        self.sharp = torch.rand((self.ROWS, self.NODES + 1, 1), generator=g).to(DEV)
        self.uniforms = torch.rand((self.ROWS, slots), generator=g).to(DEV)
        self.kw = dict(fresh=self.fresh, scale=1 / math.sqrt(d), bias=self.bias)

    def cache(self):
        return mrt_df.PagedCache(self.k, self.v, self.table, self.length, self.k_scale, self.v_scale)

    def product(self, x, w, **kw):
        codes = mrt_df.i8_quantize(x)
        y = mrt_df.i8_matmul(*codes, *w, **kw)
        self.products.append((x, codes, w, kw, y))
        return y

    def step(self):
        h, kv, d, rows = self.HEADS, self.KV, self.D, self.ROWS
        self.products = []
        there = self.slot < (self.fresh - 1)[:, None]
        drafts = torch.where(there, (self.token[:, None] * 7 + 131 * (self.slot + 1)) % self.VOCAB, -1).to(torch.int32)
        fed = torch.cat([self.token[:, None], drafts.clamp(min=0)], 1).long()
        x = self.emb[fed].view(-1, self.MODEL)
        y = self.product(x, self.w_in, dtype=self.dt).view(rows, self.NODES + 1, -1)
        self.q = y[..., :h * d].unflatten(-1, (h, d))
        self.kn, self.vn = (y[..., (h + z * kv) * d:(h + (z + 1) * kv) * d].unflatten(-1, (kv, d)) for z in range(2))
        mrt_df.paged_write(self.cache(), self.kn, self.vn, fresh=self.fresh, length_out=self.grown)
        self.out, self.lse = mrt_df.paged_attention(self.q, self.cache(), **self.kw)
        z = self.product(self.out.view(-1, h * d), self.w_back, add=x)
        logits = self.product(z, self.w_head, dtype=torch.float32).view(rows, self.NODES + 1, -1)
        self.target = (logits * 2).softmax(-1)
        # drafts that know the target more or less, so that paths of every length are accepted
        self.draft = (logits * 2 * self.sharp).softmax(-1)[:, :self.NODES]
        best = self.target[:, :self.NODES].argmax(-1).to(torch.int32)
        self.drafts = torch.where(there & (self.uniforms[:, :self.NODES] < 0.7), best, drafts)
        self.drafts = torch.where(there, self.drafts, -1)
        self.accepted, self.count, token = mrt_df.draft_verify(self.target, self.draft, self.drafts, self.uniforms)
        self.token.copy_(token)
        self.length.add_(1 + self.count)
        self.uniforms.copy_((self.uniforms * 3 + 0.37) % 1)

    def state(self):
        torch.cuda.synchronize()
        return {n: getattr(self, n).cpu().clone() for n in ("k", "v", "k_scale", "v_scale", "length", "token", "uniforms")
                if getattr(self, n) is not None}


@pytest.mark.parametrize("dtype,store", [("bf16", "i8"), ("fp32", "i8"), ("bf16", "own"), ("fp16", "own")])
def test_server_steps_against_64_bits(dtype, store):
    srv = Server(3, dtype, store)
    host = lambda t: t.cpu() if isinstance(t, torch.Tensor) else t  # noqa: E731
    lengths = srv.length.tolist()
    for _ in range(3):
        was = {"k_scale": None, "v_scale": None, "table": srv.table.cpu(), **srv.state()}
        srv.step()
        now = {"k_scale": None, "v_scale": None, **srv.state()}
        for x, codes, w, kw, y in srv.products:
            want, ws = O.quantise(x.cpu())
            assert torch.equal(codes[0].cpu(), want) and torch.equal(codes[1].cpu(), ws)
            add = kw.get("add")
            # whole numbers below 2^53: the product in fp64 on the GPU is exact
            exact = (codes[0].double() @ w[0].double().T.contiguous()) * codes[1].double()[:, None] * w[1].double()
            check_product(y, exact if add is None else exact + add.double(), add)
        want = O.paged_write(was, srv.kn.cpu(), srv.vn.cpu(), srv.fresh.cpu())
        for n in ("k", "v", "k_scale", "v_scale"):
            assert was[n] is None or same(now[n].float(), want[n].float()), n
        assert torch.equal(srv.grown.cpu(), want["length_out"])
        cache = dict(was, **{n: now[n] for n in ("k", "v", "k_scale", "v_scale")})
        check_attention(cache, dict(q=srv.q.cpu(), fresh=srv.fresh.cpu(), scale=srv.kw["scale"], bias=srv.bias.cpu()),
                        f"i8-{dtype}" if store == "i8" else dtype, (srv.out.cpu(), srv.lse.cpu()))
        paths, last = O.draft_verify(srv.target.cpu(), srv.draft.cpu(), srv.drafts.cpu(), was["uniforms"])
        assert srv.count.tolist() == [len(p) for p in paths] and now["token"].tolist() == last
        assert srv.accepted.tolist() == [p + [-1] * (srv.NODES - len(p)) for p in paths]
        lengths = [n + 1 + len(p) for n, p in zip(lengths, paths)]
        assert now["length"].tolist() == lengths


@pytest.mark.parametrize("store", ["i8", "own"])
def test_captured_servers_replay_at_once(store):
    """Two graphs with workspaces of their own, replayed side by side, with eager work on a
    third stream between the replays: bit for bit what the steps give when run one by one."""
    seeds, steps = (3, 4), 4
    want = []
    for seed in seeds:
        srv, states = Server(seed, "bf16", store), []
        for _ in range(steps):
            srv.step()
            states.append(srv.state())
        want.append(states)
    assert any(s["length"].tolist() != [2900 + i, i, 1500 + i] for states in want for i, s in enumerate(states, 1))
    srvs, graphs, streams = [Server(s, "bf16", store) for s in seeds], [], [torch.cuda.Stream() for _ in seeds]
    for srv, stream in zip(srvs, streams):
        first = srv.state()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            srv.step()  # warm, then back to the start
            for n, x in first.items():
                getattr(srv, n).copy_(x.to(DEV))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            srv.step()
        graphs.append(graph)
        torch.cuda.synchronize()
    other, aside = Server(9, "fp16", store), torch.cuda.Stream()
    aside.wait_stream(torch.cuda.current_stream())
    for i in range(steps):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(aside):
            other.step()
        for srv, states in zip(srvs, want):
            got = srv.state()
            for n, x in states[i].items():
                assert torch.equal(got[n].float(), x.float()), (i, n)


def test_the_current_device_and_stream_stay():
    """Calls go to the stream that is current, and leave it and the device as they were."""
    srv = Server(5, "bf16", "i8")
    aside = torch.cuda.Stream()
    aside.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(aside):
        srv.step()
        done = torch.cuda.Event()
        done.record()
        assert torch.cuda.current_stream() == aside and torch.cuda.current_device() == 0
    done.synchronize()
    token = srv.token.clone()
    again = Server(5, "bf16", "i8")
    again.step()
    assert torch.equal(token, again.token)
