"""Rows into cache pages and back, attention over pages and over packed prompts, against plain 64-bit forms."""
import math

import numpy as np
import pytest
import torch

import gguf_runner_b200 as g
from gguf_runner_b200.binding import AttnConfig, GgrError, KV_BF16, ROPE_ADJACENT, ROPE_NEOX, SCALE_Q_PRESCALED
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def context(hq, hkv, d, layers=1, windows=(), **more):
    return g.AttnContext(AttnConfig(n_layers=layers, n_heads=hq, n_kv_heads=hkv, head_dim=d, seq_len=8, kv_format=KV_BF16,
                                    rope_theta=1e6, swa_pattern=0, layer_windows=windows, **more))


def tables(kv_len, page, spare=2, seed=0):
    used = [-(-n // page) for n in kv_len]
    order = np.random.default_rng(seed).permutation(sum(used) + spare)
    at = np.concatenate([[0], np.cumsum(used)])
    return [order[at[i]:at[i + 1]].tolist() for i in range(len(kv_len))], sum(used) + spare


class Case:
    """Pages filled with random rows (everything else in the pool: NaN) and a batch set on them."""

    def __init__(self, hq, hkv, d, kv, dtype, page, q_len, kv_len, window=0, seed=0, layers=1, layer=0, **more):
        self.hq, self.hkv, self.d, self.kv, self.dtype, self.page = hq, hkv, d, kv, TYPES[dtype], page
        self.q_len, self.kv_len, self.window, self.layer = q_len, kv_len, window, layer
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx = context(hq, hkv, d, layers=layers, windows=(window,) * layers, **more)
        self.scale = 1.0 if more.get("scale_mode") == SCALE_Q_PRESCALED else 1.0 / math.sqrt(d)
        self.table, n_pages = tables(kv_len, page, seed=seed)
        shape = (layers, n_pages, hkv, page, d)
        q8 = kv == "q8_head"
        self.pool = [torch.full(shape, 100 if q8 else float("nan"), dtype=torch.int8 if q8 else torch.bfloat16, device="cuda") for _ in range(2)]
        self.scales = [torch.full(shape[:-1], float("nan"), device="cuda") for _ in range(2)] if q8 else [None, None]
        self.rows = []  # per sequence: k, v [key][Hkv][d] as the cache holds them
        for b, n in enumerate(kv_len):
            x = torch.randn(2, n, hkv, d, generator=gen, device="cuda")
            held = []
            for i in range(2):
                ids = torch.tensor([self.table[b][p // page] for p in range(n)], dtype=torch.long, device="cuda")
                at = torch.arange(n, device="cuda") % page
                if q8:
                    code, step = ref.quantise(x[i])
                    self.pool[i][layer, ids, :, at] = code
                    self.scales[i][layer, ids, :, at] = step
                    held.append(code.double() * step.double().unsqueeze(-1))
                else:
                    self.pool[i][layer, ids, :, at] = x[i].bfloat16()
                    held.append(x[i].bfloat16().double())
            self.rows.append(held)
        self.pages = g.Pages(self.ctx, n_pages, page, kv, *self.pool, *self.scales)
        self.batch = g.Batch(self.ctx, self.pages, dtype, max_seqs=len(kv_len), max_tokens=max(1, sum(q_len)), max_pages=max(1, sum(map(len, self.table))))
        self.batch.set(q_len, kv_len, self.table)
        self.q = torch.randn(sum(q_len), hq * d, generator=gen, device="cuda").to(self.dtype)

    def want(self):
        at, parts = 0, []
        for b, n in enumerate(self.q_len):
            q = self.q[at:at + n].view(n, self.hq, self.d)
            parts.append(ref.attention(q, *self.rows[b], self.kv_len[b] - n, self.window, self.scale))
            at += n
        return [torch.cat([p[i] for p in parts]).view(at, self.hq * self.d) for i in range(3)]

    def check(self, got):
        out, size, reach = self.want()
        err, allowed = (got.double() - out).abs(), ref.bound(self.dtype, out, size, reach)
        assert got.dtype == self.dtype and bool(torch.isfinite(got).all())
        assert bool((err <= allowed).all()), float((err / allowed).max())
        if self.dtype == torch.float32 and err.numel():  # 32-bit precision as a whole
            assert float(err.norm() / out.norm()) < 1e-6


SHAPES = [(16, 8, 128), (32, 4, 128), (40, 8, 128), (8, 4, 256), (8, 2, 64), (7, 1, 64), (4, 4, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_single_tokens(hq, hkv, d, kv, dtype):
    kv_len = [1, 2, 15, 16, 17, 130, 257, 1000]
    c = Case(hq, hkv, d, kv, dtype, 16, [1] * len(kv_len), kv_len)
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_mixed_chunks(hq, hkv, d, kv, dtype):
    q_len, kv_len = [1, 0, 5, 40, 1, 131, 2], [300, 77, 5, 333, 64, 140, 129]
    c = Case(hq, hkv, d, kv, dtype, 32, q_len, kv_len, seed=1)
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "q8_head")])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_page_sizes_and_layers(page, dtype, kv):
    c = Case(8, 2, 128, kv, dtype, page, [1, 70, 3], [page, 2 * page + 75, 700], layers=3, layer=2, seed=2)
    c.check(c.ctx.paged_attention(c.batch, 2, c.q))


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "bf16"), ("bf16", "q8_head")])
@pytest.mark.parametrize("window", [1, 16, 33, 200])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_windows(d, window, dtype, kv):
    c = Case(8, 4, d, kv, dtype, 16, [1, 50, 150, 1], [500, 300, 150, 7], window=window, seed=3)
    # pages before every window have been given back: their entries name any page
    for b, n in enumerate(c.kv_len):
        for j in range(max(0, (n - c.q_len[b] - window) // 16)):
            c.table[b][j] = c.pages.n_pages - 1
    c.batch.set(c.q_len, c.kv_len, c.table)
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))


@pytest.mark.parametrize("dtype,kv,d", [("bf16", "bf16", 128), ("f32", "bf16", 128), ("bf16", "q8_head", 128), ("bf16", "bf16", 256)])
def test_long_contexts(dtype, kv, d):
    c = Case(8, 2, d, kv, dtype, 64, [1, 3, 1], [20000, 9001, 40], seed=4)
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f32", "bf16"), ("bf16", "q8_head")])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_is_not_seen_does_not_count(d, bad, dtype, kv):
    """A later token of the chunk with values that are not finite leaves the rows before it as they are."""
    q_len, kv_len = [40, 200], [40, 260]
    clean = Case(8, 4, d, kv, dtype, 16, q_len, kv_len, seed=5)
    c = Case(8, 4, d, kv, dtype, 16, q_len, kv_len, seed=5)
    at = [21, 199]  # of sequence 0 and 1
    for b, p in enumerate(at):
        page, row = c.table[b][p // 16], p % 16
        for i in range(2):
            if kv == "bf16":
                c.pool[i][0, page, 1, row, 3] = bad
            else:
                c.scales[i][0, page, 1, row] = bad
    a, b = (x.ctx.paged_attention(x.batch, 0, x.q) for x in (clean, c))
    rows = torch.arange(a.shape[0], device="cuda")
    pos = torch.cat([torch.arange(k - n, k) for n, k in zip(q_len, kv_len)]).cuda()
    hit = torch.where(rows < q_len[0], pos >= at[0], pos >= at[1])
    heads = torch.arange(8, device="cuda") // 2 == 1
    spoilt = hit.view(-1, 1, 1) & heads.view(1, 8, 1)
    view_a, view_b = a.view(-1, 8, d), b.view(-1, 8, d)
    untouched = ~spoilt.expand_as(view_a)
    # (rows that were computed again differ in their order of sums: their own error bound)
    c.rows = clean.rows
    out, size, reach = clean.want()
    allowed = ref.bound(c.dtype, out, size, reach).view_as(view_a)
    assert bool((((view_b.double() - out.view_as(view_a)).abs() <= allowed) | ~untouched).all())
    assert bool((~torch.isfinite(view_b)[spoilt.expand_as(view_a)]).any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
@pytest.mark.parametrize("d,adjacent,rope_dim", [(128, False, 0), (128, True, 0), (64, False, 0), (256, False, 0), (128, False, 64)])
def test_append_rotates_and_stores(d, adjacent, rope_dim, kv, dtype):
    hq, hkv, page = 6, 2, 16
    q_len, kv_len = [1, 0, 19, 3], [40, 16, 19, 6000]
    ctx = context(hq, hkv, d, layers=2, rope_style=ROPE_ADJACENT if adjacent else ROPE_NEOX, rope_dim=rope_dim)
    table, n_pages = tables(kv_len, page)
    pages = g.Pages(ctx, n_pages, page, kv)
    batch = g.Batch(ctx, pages, dtype, 4, 32, 400)
    batch.set(q_len, kv_len, table)
    gen = torch.Generator(device="cuda").manual_seed(6)
    n, (qd, kd) = sum(q_len), (hq * d, hkv * d)
    wide = torch.randn(n, qd + 2 * kd + 16, generator=gen, device="cuda").to(TYPES[dtype])  # one projection's output
    q, k, v = wide[:, :qd], wide[:, qd:qd + kd], wide[:, qd + kd:qd + 2 * kd]
    before = wide.clone()
    out = torch.full((n + 2, qd), 7.0, dtype=TYPES[dtype], device="cuda")
    ctx.paged_append(batch, 1, k, v, q=q, q_out=out)
    assert torch.equal(wide, before) and bool((out[n:] == 7.0).all())
    pos = torch.cat([torch.arange(m - i, m) for i, m in zip(q_len, kv_len)]).cuda()
    rd = rope_dim or d

    def turned(x, heads):
        x = x.reshape(n, heads, d)
        return torch.cat([ref.rope(x[..., :rd], pos, rd, adjacent, 1e6), x[..., rd:].double()], -1)

    # Rotation of pairs of length at most 8 in f32, by angles brought into one turn in 64 bits: the angle, its sine and cosine, two
    # products and a sum are off by 2^-22 of that length at most each, 2^-20 in all.
    slack = torch.full((n, 1), 8 * 2.0 ** -20, dtype=torch.float64, device="cuda")
    want_q, half = turned(q, hq).view(n, qd), 2.0 ** (-8 if dtype == "bf16" else -24)
    assert bool(((out[:n].double() - want_q).abs() <= half * want_q.abs() + slack).all())
    got_k, got_v = ctx.paged_read(batch, 1, "f32")
    at = 0
    for b, m in enumerate(kv_len):
        new = slice(at + m - q_len[b], at + m)
        toks = slice(sum(q_len[:b]), sum(q_len[:b + 1]))
        want_k = turned(k, hkv)[toks].view(-1, hkv, d)
        want_v = v.reshape(n, hkv, d)[toks].double()
        for got, want in ((got_k, want_k), (got_v, want_v)):
            mine, room = got[new].view(-1, hkv, d).double(), slack[toks].unsqueeze(-1)
            if kv == "bf16":
                assert bool(((mine - want).abs() <= 2.0 ** -8 * want.abs() + room).all())
            else:  # half a step of the head, and a step of the f32 arithmetic
                step = want.abs().amax(-1, keepdim=True) / 127
                assert bool(((mine - want).abs() <= step * (0.5 + 2.0 ** -10) + 2 * room).all())
        assert not bool(got_k[at:at + m - q_len[b]].any())  # rows before the chunk: untouched (the pool was cleared)
        at += m
    other = ctx.paged_read(batch, 0, "f32")
    assert not bool(other[0].any()) and not bool(other[1].any())  # the other layer


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (256, 256)])
def test_8_bit_rows_come_back_as_their_codes(d, page, dtype):
    hkv, q_len = 3, [1, 37, 300]
    ctx = context(3, hkv, d)
    table, n_pages = tables(q_len, page)
    pages = g.Pages(ctx, n_pages, page, "q8_head")
    batch = g.Batch(ctx, pages, dtype, 3, 400, 40)
    batch.set(q_len, q_len, table)
    gen = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.randn(sum(q_len), hkv * d, generator=gen, device="cuda").to(TYPES[dtype]) for _ in range(2))
    k[5, :d] = 0.0              # a head of zeros
    k[6, d:2 * d] *= 1e-37      # too small for a scale
    k[7] *= 1e30
    v[8, 2 * d + 3] = math.nan  # one head of one row
    v[9, 1] = -math.inf
    ctx.paged_append(batch, 0, k, v)
    for out_dtype in ("f32", "bf16"):
        for got, x in zip(ctx.paged_read(batch, 0, out_dtype), (k, v)):
            code, step = ref.quantise(torch.where(torch.isfinite(x), x, torch.zeros_like(x)).view(-1, hkv, d))
            want = (code.float() * step.unsqueeze(-1)).to(TYPES[out_dtype])
            odd = ~torch.isfinite(x.view(-1, hkv, d)).all(-1, keepdim=True).expand_as(want)
            got = got.view(-1, hkv, d)
            assert bool(got[odd].isnan().all())
            assert torch.equal(torch.where(odd, torch.zeros_like(got), got), torch.where(odd, torch.zeros_like(want), want))


def test_read_into_slices_and_shared_pages():
    c = Case(4, 2, 128, "bf16", "bf16", 32, [0, 1, 0], [100, 64, 33], seed=8)
    c.table[2][0] = c.table[0][0]  # a common prefix
    c.batch.set([0, 1, 0], [100, 64, 32], c.table)
    both = torch.full((196 + 3, 2 * 256 + 8), 3.0, device="cuda")
    c.ctx.paged_read(c.batch, 0, "f32", k_out=both[:, :256], v_out=both[:, 256:512])
    for i in range(2):
        want = torch.cat([c.rows[0][i], c.rows[1][i], c.rows[0][i][:32]]).view(196, 256)
        assert torch.equal(both[:196, 256 * i:256 * i + 256].double(), want)
    assert bool((both[196:] == 3.0).all()) and bool((both[:, 512:] == 3.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_packed_prompts(hq, hkv, d, window, dtype):
    lens = [1, 7, 128, 0, 300, 33]
    n, t = sum(lens), TYPES[dtype]
    ctx = context(hq, hkv, d, windows=(window,))
    batch = g.Batch(ctx, None, dtype, 6, 600)
    batch.set(lens)
    gen = torch.Generator(device="cuda").manual_seed(9)
    wide = torch.randn(n, (hq + 2 * hkv) * d, generator=gen, device="cuda").to(t)
    q, k, v = wide[:, :hq * d], wide[:, hq * d:(hq + hkv) * d], wide[:, (hq + hkv) * d:]
    out = torch.full((n + 5, hq * d), 7.0, dtype=t, device="cuda")
    ctx.packed_attention(batch, 0, q, k, v, out=out)
    assert bool((out[n:] == 7.0).all())
    at, parts = 0, []
    for m in lens:
        rows = [x[at:at + m].reshape(m, h, d) for x, h in ((q, hq), (k, hkv), (v, hkv))]
        parts.append(ref.attention(*rows, 0, window, 1 / math.sqrt(d)))
        at += m
    want, size, reach = (torch.cat([p[i] for p in parts]).view(n, hq * d) for i in range(3))
    err, allowed = (out[:n].double() - want).abs(), ref.bound(t, want, size, reach)
    assert bool((err <= allowed).all()), float((err / allowed).max())
    if dtype == "f32":
        assert float(err.norm() / want.norm()) < 1e-6


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_packed_prompts_do_not_touch_each_other(dtype):
    lens, t = [33, 50, 20], TYPES[dtype]
    ctx = context(8, 2, 128)
    batch = g.Batch(ctx, None, dtype, 3, 200)
    batch.set(lens)
    gen = torch.Generator(device="cuda").manual_seed(10)
    q, k, v = (torch.randn(sum(lens), h * 128, generator=gen, device="cuda").to(t) for h in (8, 2, 2))
    want = ctx.packed_attention(batch, 0, q, k, v).clone()
    k[33:83], v[33:83] = math.nan, math.inf
    got = ctx.packed_attention(batch, 0, q, k, v)
    assert torch.equal(got[:33], want[:33]) and torch.equal(got[83:], want[83:])


def test_a_step_as_a_server_runs_it():
    """Two layers, prompts in chunks beside token steps, appended and attended, against the dense cache of the same context."""
    cfg = dict(layers=2, hq=8, hkv=2, d=128)
    ctx = context(cfg["hq"], cfg["hkv"], cfg["d"], layers=2)
    dense = g.AttnContext(AttnConfig(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, seq_len=400, max_batch=3, kv_format=KV_BF16,
                                     rope_theta=1e6, swa_pattern=0))
    norm = np.linspace(0.8, 1.2, 128).astype(np.float32)
    for x in (ctx, dense):
        x.set_layer_fixups(1, q_norm=norm, k_norm=norm[::-1].copy(), eps=1e-6)
    table, n_pages = tables([400] * 3, 16)
    pages = g.Pages(ctx, n_pages, 16)
    batch = g.Batch(ctx, pages, "f32", 3, 400, 3 * 25)
    gen = torch.Generator(device="cuda").manual_seed(11)
    have = [0, 0, 0]
    for q_len in ([100, 0, 0], [1, 64, 0], [1, 64, 200], [1, 1, 1], [1, 1, 1]):
        have = [h + n for h, n in zip(have, q_len)]
        batch.set(q_len, have, table)
        for layer in range(2):
            q, k, v = (torch.randn(sum(q_len), h * 128, generator=gen, device="cuda") for h in (8, 2, 2))
            turned = ctx.paged_append(batch, layer, k, v, q=q)
            got = ctx.paged_attention(batch, layer, turned)
            at = 0
            for b, n in enumerate(q_len):
                if n:
                    s = slice(at, at + n)
                    want = dense.prefill(layer, have[b] - n, q[s].contiguous(), k[s].contiguous(), v[s].contiguous(), seq=b)
                    assert float((got[s] - want).abs().max()) < 2e-2  # the dense path rounds q and the weights to bf16
                at += n


def test_captured_steps_follow_the_plan():
    c = Case(32, 8, 128, "bf16", "bf16", 16, [1, 1, 1], [700, 30, 1], seed=12)
    big = Case(32, 8, 128, "bf16", "bf16", 16, [1, 1, 1], [900, 900, 900], seed=13)
    c.close = None
    lens = [[700, 30, 1], [900, 899, 64], [1, 1, 1]]
    ctx, batch = big.ctx, big.batch
    out = torch.empty_like(big.q)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    k, v = (torch.randn(3, 8 * 128, device="cuda").bfloat16() for _ in range(2))
    with torch.cuda.stream(side):
        batch.set([1, 1, 1], lens[0], big.table)
        ctx.paged_attention(batch, 0, big.q, out=out)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            ctx.paged_append(batch, 0, k, v)
            ctx.paged_attention(batch, 0, big.q, out=out)
        for kv in lens:
            batch.set([1, 1, 1], kv, big.table)
            out.zero_()
            graph.replay()
            side.synchronize()
            got = out.clone()
            again = torch.empty_like(out)
            ctx.paged_append(batch, 0, k, v)
            ctx.paged_attention(batch, 0, big.q, out=again)
            side.synchronize()
            assert torch.equal(got, again)
            rows = ctx.paged_read(batch, 0, "bf16")[0]
            side.synchronize()
            assert torch.equal(rows[kv[0] - 1], k[0])
        with pytest.raises(GgrError):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                batch.set([1, 1, 1], lens[0], big.table)


@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
@pytest.mark.parametrize("d", [128, 256])
def test_cut_chunks(d, kv):
    """Few rows and many keys: items are cut along the keys and merged; one row of a piece is not finite."""
    c = Case(8, 2, d, kv, "bf16", 64, [70, 1, 33], [7000, 50, 3001], seed=16)
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))
    first = c.ctx.paged_attention(c.batch, 0, c.q).clone()
    for _ in range(3):
        assert torch.equal(c.ctx.paged_attention(c.batch, 0, c.q), first)


def test_8_bit_rows_beyond_f16():
    """Values that the f16 operands of a chunk cannot hold: those rows are computed again in f32."""
    c = Case(8, 2, 128, "q8_head", "bf16", 16, [40], [90], seed=17)
    for i, by in enumerate((3e4, 5e3)):
        page, row = c.table[0][60 // 16], 60 % 16
        c.scales[i][0, page, 1, row] *= by
        c.rows[0][i][60, 1] *= float(torch.tensor(by, dtype=torch.float32))
    got = c.ctx.paged_attention(c.batch, 0, c.q)
    out, size, reach = c.want()
    # (scores of up to 1e5: only the largest weight counts, and an f32 score is off by 2^-20 of its reach)
    allowed = ref.bound(c.dtype, out, size, reach)
    assert bool(((got.double() - out).abs() <= allowed).all())


def test_many_sequences():
    lens = [1 + (i * 37) % 60 for i in range(300)]
    q_len = [min(n, 1 + i % 3) for i, n in enumerate(lens)]
    for kv, dtype in (("bf16", "bf16"), ("q8_head", "f32")):
        c = Case(4, 2, 64, kv, dtype, 16, q_len, lens, seed=18)
        c.check(c.ctx.paged_attention(c.batch, 0, c.q))


def test_plans_and_streams_do_not_meet():
    """Two plans of one context in turn, one of them on a side stream: nothing is shared but the pool."""
    c = Case(32, 8, 128, "bf16", "bf16", 16, [1, 40], [3000, 700], seed=19)
    want = c.ctx.paged_attention(c.batch, 0, c.q).clone()
    other = g.Batch(c.ctx, c.pages, "bf16", 2, 41, 300)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other.set([1, 1], [900, 600], c.table)
    small = c.q[:2].contiguous()
    torch.cuda.synchronize()
    ref_small = None
    for _ in range(3):
        a = c.ctx.paged_attention(c.batch, 0, c.q)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            b = c.ctx.paged_attention(other, 0, small)
        torch.cuda.synchronize()
        assert torch.equal(a, want)
        ref_small = b.clone() if ref_small is None else ref_small
        assert torch.equal(b, ref_small)


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("bf16", "q8_head"), ("f32", "q8_head")])
def test_captured_plans_keep_to_their_kernels(dtype, kv):
    """A plan with captured token steps still serves chunks (with the kernels of the steps); captured chunks are replayed with
    single tokens, other lengths and cuts."""
    for start, later in (([1, 1], [40, 150]), ([40, 150], [1, 2])):
        c = Case(8, 2, 128, kv, dtype, 16, [40, 150], [2000, 700], seed=20)
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        out = torch.empty_like(c.q)
        with torch.cuda.stream(side):
            c.batch.set(start, c.kv_len, c.table)
            c.ctx.paged_attention(c.batch, 0, c.q, out=out)
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                c.ctx.paged_attention(c.batch, 0, c.q, out=out)
            for q_len in (later, start):
                c.batch.set(q_len, c.kv_len, c.table)
                n = sum(q_len)
                all_q, c.q_len = c.q, q_len
                graph.replay()
                side.synchronize()
                c.q = all_q[:n]
                c.check(out[:n])
                c.check(c.ctx.paged_attention(c.batch, 0, c.q))
                side.synchronize()
                c.q = all_q
        with pytest.raises(GgrError), torch.cuda.stream(side):  # nothing to capture
            c.batch.set([0, 0], c.kv_len, c.table)
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                c.ctx.paged_attention(c.batch, 0, c.q, out=out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_packed_prompts(dtype):
    t, ctx = TYPES[dtype], context(8, 2, 128)
    batch = g.Batch(ctx, None, dtype, 4, 300)
    gen = torch.Generator(device="cuda").manual_seed(21)
    q, k, v = (torch.randn(300, h * 128, generator=gen, device="cuda").to(t) for h in (8, 2, 2))
    out = torch.empty_like(q)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        batch.set([100, 60])
        ctx.packed_attention(batch, 0, q, k, v, out=out)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            ctx.packed_attention(batch, 0, q, k, v, out=out)
        with pytest.raises(ValueError):  # a replay may find more rows than this
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                ctx.packed_attention(batch, 0, q[:160], k, v, out=out)
        for lens in ([7, 250, 1, 42], [3], [150, 150]):
            batch.set(lens)
            out.fill_(7.0)
            graph.replay()
            side.synchronize()
            n = sum(lens)
            assert bool((out[n:] == 7.0).all())
            fresh = g.Batch(ctx, None, dtype, 4, 300)
            fresh.set(lens)
            want = ctx.packed_attention(fresh, 0, q, k, v)[:n]
            side.synchronize()
            assert float((out[:n].float() - want.float()).abs().max()) <= (2.0 ** -7 * 4 if dtype == "bf16" else 1e-5)


def test_window_layers_rotate_by_their_own_theta():
    ctx = g.AttnContext(AttnConfig(n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128, seq_len=8, kv_format=KV_BF16, rope_theta=1e6,
                                   rope_theta_swa=1e4, swa_theta_on_window_layers=1, layer_windows=(64, 0)))
    pages = g.Pages(ctx, 8, 16)
    batch = g.Batch(ctx, pages, "f32", 1, 10, 8)
    batch.set([10], [100], [list(range(7))])
    q, k, v = (torch.randn(10, h * 128, device="cuda") for h in (4, 2, 2))
    pos = torch.arange(90, 100, device="cuda")
    for layer, theta in ((0, 1e4), (1, 1e6)):
        got = ctx.paged_append(batch, layer, k, v, q=q)
        want = ref.rope(q.view(10, 4, 128), pos, 128, False, theta).view(10, 512)
        assert float((got.double() - want).abs().max()) < 8 * 2.0 ** -20
        same = q.clone()
        assert ctx.paged_append(batch, layer, k, v, q=same, q_out=same) is same and torch.equal(same, got)


def test_pools_beyond_32_bit_offsets():
    """Pages whose rows lie more than 2^32 elements into the pool."""
    n_pages, page, hkv, d = 20000, 256, 8, 128
    pool = [torch.empty(1, n_pages, hkv, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ctx = context(8, hkv, d)
    pages = g.Pages(ctx, n_pages, page, "bf16", *pool)
    batch = g.Batch(ctx, pages, "bf16", 2, 400, 10)
    q_len, kv_len = [300, 1], [300, 1]
    table = [[19999, 0], [19000]]
    gen = torch.Generator(device="cuda").manual_seed(22)
    q, k, v = (torch.randn(301, h * d, generator=gen, device="cuda").bfloat16() for h in (8, hkv, hkv))
    batch.set(q_len, kv_len, table)
    ctx.paged_append(batch, 0, k, v)
    assert torch.equal(pool[0][0, 19999, :, :256].transpose(0, 1).reshape(256, -1), k[:256])
    got_k, got_v = ctx.paged_read(batch, 0, "bf16")
    assert torch.equal(got_k, k) and torch.equal(got_v, v)
    got = ctx.paged_attention(batch, 0, q)
    out, size, reach = (x.view(300, -1) for x in ref.attention(q[:300].view(300, 8, d), k[:300].view(300, hkv, d), v[:300].view(300, hkv, d), 0, 0, d ** -0.5))
    assert bool(((got[:300].double() - out).abs() <= ref.bound(torch.bfloat16, out, size, reach)).all())
    assert torch.equal(got[300], v[300].view(hkv, d).reshape(-1))


@pytest.mark.parametrize("d,kv,dtype", [(128, "bf16", "bf16"), (128, "q8_head", "bf16"), (64, "q8_head", "f32"), (256, "bf16", "bf16")])
def test_launches_keep_their_order(d, kv, dtype):
    """Appends over the same pages, attention, reads and foreign kernels behind each other, against the same step by step."""
    c = Case(8, 2, d, kv, dtype, 16, [1, 60, 2], [900, 300, 33], seed=23)
    gen = torch.Generator(device="cuda").manual_seed(24)
    steps = [torch.randn(3, 63, 8 * d, generator=gen, device="cuda").to(c.dtype) for _ in range(6)]

    arrays = [x for x in c.pool + c.scales if x is not None]
    start = [x.clone() for x in arrays]

    def play(wait):
        got = []
        for x, s in zip(arrays, start):
            x.copy_(s)
        for i, x in enumerate(steps):
            # a plan of its own for every step: nothing may be read of the one before
            kv_len = [c.kv_len[0] - 61 * i, c.kv_len[1] - 17 * i, c.kv_len[2] - i]
            c.batch.set(c.q_len, kv_len, c.table)
            q = x[0] * 1.0  # a kernel of torch's in front
            k, v = x[1, :, :2 * d] * 1.0, x[2, :, :2 * d] * 1.0
            wait()
            turned = c.ctx.paged_append(c.batch, 0, k, v, q=q)
            wait()
            out = c.ctx.paged_attention(c.batch, 0, turned)
            wait()
            c.ctx.paged_append(c.batch, 0, v, k)  # over the rows that were just read
            wait()
            rows = c.ctx.paged_read(c.batch, 0, dtype)
            wait()
            again = c.ctx.paged_attention(c.batch, 0, turned)
            wait()
            turned.zero_()
            got += [out, again, *(r[torch.isfinite(r)] for r in rows)]
        torch.cuda.synchronize()
        return got

    want = play(torch.cuda.synchronize)
    for _ in range(3):
        for a, b in zip(play(lambda: None), want):
            assert torch.equal(a, b)


def test_results_repeat_bit_for_bit():
    c = Case(32, 4, 128, "bf16", "bf16", 32, [1] * 5 + [60], [5000, 40, 900, 2500, 1, 300], seed=14)
    first = c.ctx.paged_attention(c.batch, 0, c.q).clone()
    for _ in range(5):
        assert torch.equal(c.ctx.paged_attention(c.batch, 0, c.q), first)


def test_more_heads_than_a_query_tile_has_rows():
    c = Case(160, 1, 64, "bf16", "bf16", 16, [1, 9], [70, 300], seed=25)
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))


def test_closed_handles_are_refused():
    c = Case(4, 2, 64, "bf16", "bf16", 16, [1], [5])
    c.ctx.close()
    with pytest.raises(ValueError):
        c.batch.set([1], [5], c.table)
    with pytest.raises(GgrError):
        c.ctx.paged_attention(c.batch, 0, c.q)


def test_prescaled_queries():
    c = Case(8, 4, 256, "bf16", "bf16", 16, [1, 30], [90, 100], seed=15, scale_mode=SCALE_Q_PRESCALED)
    c.q /= 16.0
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))


def test_refusals():
    ctx, other = context(8, 2, 128), context(8, 2, 128)
    for bad in (dict(n_pages=0, page_size=16), dict(n_pages=4, page_size=8), dict(n_pages=4, page_size=48), dict(n_pages=4, page_size=512)):
        with pytest.raises(GgrError):
            g.Pages(ctx, **bad)
    with pytest.raises(ValueError):
        g.Pages(ctx, 4, 16, "q4")
    with pytest.raises(ValueError):
        g.Pages(ctx, 4, 16, "bf16", k=torch.zeros(10, device="cuda", dtype=torch.bfloat16), v=None)
    with pytest.raises(GgrError):  # half of a pool
        g.Pages(ctx, 4, 16, "bf16", k=torch.zeros(1, 4, 2, 16, 128, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(GgrError):
        g.Pages(context(8, 2, 96), 4, 16)
    pages = g.Pages(ctx, 8, 16)
    with pytest.raises(GgrError):
        g.Batch(other, pages, "bf16", 1, 1, 1)
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(GgrError):
            g.Batch(ctx, pages, "bf16", *bad)
    batch = g.Batch(ctx, pages, "bf16", 2, 20, 8)
    q, k, v = (torch.zeros(20, h * 128, device="cuda", dtype=torch.bfloat16) for h in (8, 2, 2))
    with pytest.raises(GgrError):  # not set
        ctx.paged_attention(batch, 0, q)
    for q_len, kv_len, table in (([1, 1, 1], [1, 1, 1], [[0], [1], [2]]), ([2], [1], [[0]]), ([-1], [1], [[0]]), ([21], [21], [[0, 1]]), ([1], [1], [[8]]),
                                 ([1], [1], [[-1]]), ([1, 1], [20, 20], [[0, 1], [2, 1]]), ([17], [33], [[0, 1, 1]])):
        with pytest.raises(GgrError):
            batch.set(q_len, kv_len, table)
    with pytest.raises(ValueError):
        batch.set([1], [40], [[0, 1]])
    with pytest.raises(GgrError):  # a plan that could not be set is not in force
        ctx.paged_attention(batch, 0, q)
    batch.set([1, 2], [20, 30], [[0, 1], [2, 3]])
    with pytest.raises(GgrError):
        ctx.paged_attention(batch, 1, q)
    with pytest.raises(GgrError):
        other.paged_attention(batch, 0, q)
    with pytest.raises(GgrError):
        ctx.packed_attention(batch, 0, q, k, v)
    with pytest.raises(ValueError):
        ctx.paged_attention(batch, 0, q.float())
    with pytest.raises(ValueError):
        ctx.paged_attention(batch, 0, q.cpu())
    with pytest.raises(ValueError):
        ctx.paged_attention(batch, 0, q[:2])
    with pytest.raises(ValueError):
        ctx.paged_attention(batch, 0, q.T.contiguous().T)
    with pytest.raises(ValueError):  # one row for all tokens
        ctx.paged_attention(batch, 0, q[:1].expand(20, 1024))
    with pytest.raises(ValueError):
        batch.set([1], [1], [[2 ** 32]])
    with pytest.raises(ValueError):
        batch.set([1.5], [2], [[0]])
    with pytest.raises(GgrError):  # rows off the 16-byte grid
        ctx.paged_attention(batch, 0, torch.zeros(20, 1025, device="cuda", dtype=torch.bfloat16)[:, 1:])
    packed = g.Batch(ctx, None, "bf16", 2, 20)
    with pytest.raises(GgrError):
        packed.set([3], [4])
    packed.set([3, 4])
    with pytest.raises(GgrError):
        ctx.paged_read(packed, 0)
    ctx.set_media_blocks([], 0)
    plan = g.RopePositionPlan()
    plan.append_text(4)
    ctx.set_position_plan(plan)
    with pytest.raises(GgrError):
        ctx.paged_append(batch, 0, k, v, q=q)
