"""Where the paged operators can go wrong: values that are not finite, rows and scales at the ends of their ranges, empty steps,
plans that are refused, closed or captured, against plain 64-bit forms."""
import math

import pytest
import torch

import gguf_runner_b200 as g
from gguf_runner_b200.binding import GgrError
from tests import paged_reference as ref
from tests.test_gpu_paged import TYPES, Case, context, tables

pytestmark = pytest.mark.gpu


def without(case, seq, key):
    """The 64-bit result, as `ref.attention` gives it, of sequence `seq` with key `key`, which all its rows see, left out."""
    at, n = sum(case.q_len[:seq]), case.q_len[seq]
    k, v = (torch.cat([x[:key], x[key + 1:]]) for x in case.rows[seq])
    return ref.attention(case.q[at:at + n].view(n, case.hq, case.d), k, v, case.kv_len[seq] - n - 1, 0, case.scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,bad", [("bf16", math.nan), ("bf16", math.inf), ("bf16", -math.inf), ("q8_head", math.nan)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_key_that_is_not_finite_counts_wherever_it_stands(d, kv, bad, dtype):
    """One element of one key of KV head 1, at every residue of 8: a score of NaN or +inf makes the rows of its heads NaN, one of
    -inf has weight 0; the other KV head is left as it is."""
    c = Case(4, 2, d, kv, dtype, 16, [150] * 8, [300] * 8, seed=31)
    c.q.view(-1, 4, d)[:, :, 0] = 1.0
    for b in range(8):
        page, row = c.table[b][(96 + b) // 16], (96 + b) % 16
        if kv == "bf16":
            c.pool[0][0, page, 1, row, 0] = bad
        else:
            c.scales[0][0, page, 1, row] = bad
    got = c.ctx.paged_attention(c.batch, 0, c.q).view(8, 150, 4, d)
    out, size, reach = (x.view(8, 150, 4, d) for x in c.want())
    off = (got.double() - out).abs() <= ref.bound(c.dtype, out, size, reach)
    assert bool(off[:, :, :2].all())
    for b in range(8):
        mine = got[b, :, 2:]
        if bad != -math.inf:
            assert bool(mine.isnan().all()), (b, float(mine.isnan().double().mean()))
        else:
            w, size, reach = without(c, b, 96 + b)
            ok = (got[b].double() - w).abs() <= ref.bound(c.dtype, w, size, reach)
            assert bool(ok[:, 2:].all()), b


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_nan_key_of_packed_prompts_counts_wherever_it_stands(d, dtype):
    lens, t = [200] * 8, TYPES[dtype]
    ctx = context(4, 2, d)
    batch = g.Batch(ctx, None, dtype, 8, 1600)
    batch.set(lens)
    gen = torch.Generator(device="cuda").manual_seed(32)
    q, k, v = (torch.randn(1600, h, d, generator=gen, device="cuda").to(t) for h in (4, 2, 2))
    spoilt = k.clone()
    for b in range(8):
        spoilt[200 * b + 96 + b, 1, 5] = math.nan
    got = ctx.packed_attention(batch, 0, q.view(1600, -1), spoilt.view(1600, -1), v.view(1600, -1)).view(8, 200, 4, d)
    for b in range(8):
        s = slice(200 * b, 200 * b + 200)
        out, size, reach = ref.attention(q[s], k[s], v[s], 0, 0, 1 / math.sqrt(d))
        ok = (got[b].double() - out).abs() <= ref.bound(t, out, size, reach)
        assert bool(ok[:, :2].all()) and bool(ok[:96 + b].all())
        assert bool(got[b, 96 + b:, 2:].isnan().all()), b


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_first_score_of_minus_infinity(d, n, dtype):
    """The first key scores -inf and a later token's value is not finite: the rows in between see the one with weight 0 and the
    other not at all."""
    c = Case(4, 2, d, "bf16", dtype, 16, [n], [n], seed=33)
    c.q.view(n, 4, d)[:, :, 0] = 1.0
    c.pool[0][0, c.table[0][0], 1, 0, 0] = -math.inf
    c.pool[1][0, c.table[0][1], 1, 5, 3] = math.nan  # position 21
    got = c.ctx.paged_attention(c.batch, 0, c.q).view(n, 4, d)
    k, v = (x[1:] for x in c.rows[0])
    out, size, reach = ref.attention(c.q.view(n, 4, d)[1:], k, v, 0, 0, c.scale)
    ok = (got[1:].double() - out).abs() <= ref.bound(c.dtype, out, size, reach)
    heads = got[:, 2:]
    assert bool(ok[:20, 2:].all()), float(heads[1:21].isnan().double().mean())
    assert bool(heads[21:, :, 3].isnan().all())
    ok[:, :, 3] = True
    assert bool(ok[20:, 2:].all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [20, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_whose_scores_are_all_minus_infinity(d, n, dtype):
    """No key has a weight: 0 / 0, as the softmax of such a row is, and not the mean or zero."""
    c = Case(4, 2, d, "bf16", dtype, 16, [n], [n], seed=39)
    c.q.view(n, 4, d)[:, :, 0] = 1.0
    c.pool[0][0, c.table[0][0], 1, :9, 0] = -math.inf
    got = c.ctx.paged_attention(c.batch, 0, c.q).view(n, 4, d)
    out, size, reach = ref.attention(c.q.view(n, 4, d)[9:], *(x[9:] for x in c.rows[0]), 0, 0, c.scale)
    assert bool(got[:9, 2:].isnan().all())
    assert bool(((got[9:].double() - out).abs() <= ref.bound(c.dtype, out, size, reach))[:, 2:].all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pieces_whose_scores_are_all_minus_infinity(d, dtype):
    """Few rows and many keys, cut along the keys: what lies in the first half has no weight."""
    c = Case(4, 2, d, "bf16", dtype, 64, [70], [7000], seed=40)
    c.q.view(70, 4, d)[:, :, 0] = 1.0
    for p in range(0, 3520, 64):
        c.pool[0][0, c.table[0][p // 64], 1, :, 0] = -math.inf
    got = c.ctx.paged_attention(c.batch, 0, c.q).view(70, 4, d)
    out, size, reach = ref.attention(c.q.view(70, 4, d), *(x[3520:] for x in c.rows[0]), 6930 - 3520, 0, c.scale)
    assert bool(((got.double() - out).abs() <= ref.bound(c.dtype, out, size, reach))[:, 2:].all())


@pytest.mark.parametrize("step", [dict(q_len=[9, 1], kv_len=[9, 1]), dict(q_len=[1] * 3, kv_len=[1] * 3), dict(q_len=[-1, 1], kv_len=[1, 1]),
                                  dict(q_len=[1, 1], kv_len=[1, 1], page_table=[[99], [0]])])
def test_a_refused_step_does_not_leave_the_one_before_in_force(step):
    """Whoever goes on has other rows than those of the step before: every call is refused until a step has been set."""
    c = Case(4, 2, 64, "bf16", "bf16", 16, [2, 3], [20, 40], seed=41)
    want = c.ctx.paged_attention(c.batch, 0, c.q)
    packed = g.Batch(c.ctx, None, "bf16", 2, 5)
    packed.set([2, 3])
    k = torch.zeros(5, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(GgrError):
        c.batch.set(**{"page_table": [[0], [1], [2]][:len(step["q_len"])], **step})
    if "page_table" not in step:
        with pytest.raises(GgrError):
            packed.set(step["q_len"])
        with pytest.raises(GgrError):
            c.ctx.packed_attention(packed, 0, c.q, k, k)
    for call in (lambda: c.ctx.paged_attention(c.batch, 0, c.q), lambda: c.ctx.paged_append(c.batch, 0, k, k), lambda: c.ctx.paged_read(c.batch, 0)):
        with pytest.raises(GgrError):
            call()
    c.batch.set(c.q_len, c.kv_len, c.table)
    assert torch.equal(c.ctx.paged_attention(c.batch, 0, c.q), want)


def test_a_pool_outlives_the_plans_on_it():
    """A closed pool's plans are refused by every call; its memory is there until the last of them is closed."""
    ctx = context(8, 8, 128, layers=4)
    start = torch.cuda.mem_get_info()[0]
    pages = g.Pages(ctx, 1000, 256)  # 2 x 2 GB
    plans = [g.Batch(ctx, pages, "bf16", 1, 4, 2) for _ in range(2)]
    k, q = (torch.zeros(4, h * 128, dtype=torch.bfloat16, device="cuda") for h in (8, 8))
    for p in plans:
        p.set([4], [4], [[7]])
        ctx.paged_append(p, 0, k, k)
    pages.close()
    pages.close()
    for call in (lambda p: p.set([4], [4], [[7]]), lambda p: ctx.paged_append(p, 0, k, k), lambda p: ctx.paged_attention(p, 0, q),
                 lambda p: ctx.paged_read(p, 0)):
        for p in plans:
            with pytest.raises((ValueError, GgrError)):
                call(p)
    with pytest.raises(ValueError):
        g.Batch(ctx, pages, "bf16", 1, 4, 2)
    with pytest.raises(GgrError):
        pages.device_ptrs()
    torch.cuda.synchronize()
    plans[0].close()
    assert start - torch.cuda.mem_get_info()[0] > 2 << 30
    plans[1].close()
    assert start - torch.cuda.mem_get_info()[0] < 1 << 30


def test_a_captured_read_has_room_for_the_longest_step():
    c = Case(4, 2, 64, "bf16", "bf16", 16, [1, 1], [20, 40], seed=36)
    most = 5 * 16  # the plan has room for five pages
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    small, large = (torch.zeros(2, n, 128, device="cuda") for n in (60, most))
    with torch.cuda.stream(side):
        c.batch.set([0, 0], [20, 10], c.table)
        c.ctx.paged_read(c.batch, 0, "f32", *small)
        side.synchronize()
        with pytest.raises(ValueError):  # a replay may find more rows than this
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                c.ctx.paged_read(c.batch, 0, "f32", *small)
        with torch.cuda.graph(graph, stream=side):
            k, v = c.ctx.paged_read(c.batch, 0, "f32", *large)
            own = c.ctx.paged_read(c.batch, 0, "f32")
        assert own[0].shape == own[1].shape == (most, 128)
        c.batch.set([1, 1], [20, 40], c.table)
        graph.replay()
        side.synchronize()
        for i, got in enumerate((k, v)):
            want = torch.cat([r[i] for r in c.rows]).view(60, 128)
            assert torch.equal(got[:60].double(), want) and not bool(got[60:].any()) and torch.equal(own[i][:60], got[:60])


def device_time(call, n=3):
    """Milliseconds of a call on the device."""
    call()
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(n):
        call()
    stop.record()
    stop.synchronize()
    return start.elapsed_time(stop) / n


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_value_that_is_not_finite_in_cut_rows(d, kv, dtype):
    """Chunks and a single token over long texts, cut along their keys: a later token's value shows in the rows that see it, in the
    elements that it spoils, and nowhere else."""
    q_len, kv_len, at = [70, 1, 33], [7000, 9000, 3001], [6950, 8999, 2990]
    c = Case(8, 2, d, kv, dtype, 64, q_len, kv_len, seed=42)
    for b, p in enumerate(at):
        page, row = c.table[b][p // 64], p % 64
        if kv == "bf16":
            c.pool[1][0, page, 1, row, 3] = math.nan
        else:
            c.scales[1][0, page, 1, row] = math.nan
    got = c.ctx.paged_attention(c.batch, 0, c.q).view(-1, 8, d)
    out, size, reach = (x.view(-1, 8, d) for x in c.want())
    ok = (got.double() - out).abs() <= ref.bound(c.dtype, out, size, reach)
    pos = torch.cat([torch.arange(k - n, k) for n, k in zip(q_len, kv_len)]).cuda()
    seen = pos >= torch.cat([torch.full((n,), p) for n, p in zip(q_len, at)]).cuda()
    spoilt = torch.zeros_like(ok)
    spoilt[seen, 4:, 3 if kv == "bf16" else slice(None)] = True
    assert bool(ok[~spoilt].all()) and bool(got[spoilt].isnan().all())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_values_in_long_texts(d):
    """Values that the f16 operands of 8-bit chunks cannot hold: the rows that see them are right, and the call ends in its time."""
    c = Case(8, 2, d, "q8_head", "bf16", 64, [150], [12000], seed=43)
    usual = device_time(lambda: c.ctx.paged_attention(c.batch, 0, c.q))
    c.scales[1][0, c.table[0][2], 1, 5] *= 2000.0
    c.rows[0][1][133, 1] *= 2000.0
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))
    took = device_time(lambda: c.ctx.paged_attention(c.batch, 0, c.q))
    # (one key after the other, a single row took 14 to 52 ms)
    assert took < 12.0, (took, usual)


def test_waits_outlast_rows_that_are_computed_again():
    """A chunk behind 300000 8-bit keys with one value beyond f16, in front of a long prompt: its rows take longer than any wait of
    their CTA is allowed to, and neither they nor the prompt's rows, whose items come behind them, are lost."""
    heads, d, page, q_len, kv_len = 8, 64, 256, [300, 38144], [300000, 38144]
    ctx = context(heads, heads, d)
    used = [-(-n // page) for n in kv_len]
    gen = torch.Generator(device="cuda").manual_seed(44)
    pool = [torch.randint(-127, 128, (1, sum(used), heads, page, d), generator=gen, device="cuda", dtype=torch.int8) for _ in range(2)]
    scales = [torch.full((1, sum(used), heads, page), 1 / 64, device="cuda") for _ in range(2)]
    scales[1][0, 0, 1, 7] = 20.0
    pages = g.Pages(ctx, sum(used), page, "q8_head", *pool, *scales)
    batch = g.Batch(ctx, pages, "bf16", 2, sum(q_len), sum(used))
    batch.set(q_len, kv_len, [list(range(used[0])), list(range(used[0], sum(used)))])
    q = torch.randn(sum(q_len), heads * d, generator=gen, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    ctx.paged_attention(batch, 0, q, out=out)
    took = device_time(lambda: ctx.paged_attention(batch, 0, q, out=out), 1)
    for b, toks in ((0, (0, 100, 299)), (1, (0, 255, 256, 20000, 38143))):
        of = slice(0, used[0]) if b == 0 else slice(used[0], None)
        for h in (0, 1, 7):
            k, v = (pool[i][0, of, h].reshape(-1, 1, d).double() * scales[i][0, of, h].reshape(-1, 1, 1).double() for i in range(2))
            for t in toks:
                n, row = kv_len[b] - q_len[b] + t + 1, t + b * q_len[0]
                want, size, reach = ref.attention(q[row].view(1, heads, d)[:, h:h + 1], k[:n], v[:n], n - 1, 0, 1 / math.sqrt(d))
                got = out[row].view(heads, d)[h].double()
                assert bool(((got - want[0, 0]).abs() <= ref.bound(torch.bfloat16, want, size, reach)[0, 0]).all()), (b, h, t)
    assert bool(torch.isfinite(out).all()) and not bool((out.view(-1, heads, d) == 7.0).all(-1).any())
    assert took > 1000.0, took  # (long enough to show it)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_zeros_over_8_bit_pages(d, dtype):
    """Rows of q that are zero or next to it, uncut and cut: every key counts the same, and they cost what others cost."""
    c = Case(8, 2, d, "q8_head", dtype, 16, [3, 1, 2], [40, 12000, 7], seed=34)
    usual = device_time(lambda: c.ctx.paged_attention(c.batch, 0, c.q))
    rows = c.q.view(6, 8, d)
    rows[0], rows[3, :3], rows[1, 2], rows[5, 7], rows[3, 5] = 0.0, 0.0, 1e-38, 1e-30, 1e-37
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))
    took = device_time(lambda: c.ctx.paged_attention(c.batch, 0, c.q))
    assert took < 5 * usual, (took, usual)  # (one row again, key by key, would take hundreds of times as long)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_small_weights_over_8_bit_pages(d):
    """One key has a weight of 1 and 20000 others 2^-26 of it, which together make 3e-4 of the sum, and all of the result."""
    n, gap = 20150, 26 * math.log(2.0)
    c = Case(4, 2, d, "q8_head", "bf16", 64, [150], [n], seed=35)
    c.q.fill_(1.0)
    high = 2.0
    low = high - gap / math.sqrt(d)  # q . k / sqrt(d) = sqrt(d) x for a key of elements x
    rows = torch.full((2, n), low, device="cuda")
    rows[0, 0], rows[1], rows[1, 0] = high, 1.0, 0.0
    for i in range(2):
        for p in range(n):
            page, row = c.table[0][p // 64], p % 64
            c.pool[i][0, page, :, row] = 127
            c.scales[i][0, page, :, row] = rows[i, p] / 127
        step = (rows[i] / 127).double()
        c.rows[0][i] = (127 * step).view(n, 1, 1).expand(n, 2, d).contiguous()
    c.check(c.ctx.paged_attention(c.batch, 0, c.q))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_steps_without_new_tokens(dtype):
    c = Case(4, 2, 64, "bf16", dtype, 16, [1, 1], [20, 40], seed=37)
    none = [torch.empty(0, h * 64, dtype=c.dtype, device="cuda") for h in (4, 2, 2)]
    for q_len, kv_len, table in (([0, 0], [20, 40], c.table), ([0, 0], [0, 0], [[], []]), ([], [], [])):
        c.batch.set(q_len, kv_len, table)
        assert c.ctx.paged_append(c.batch, 0, none[1], none[2], q=none[0]).shape == (0, 256)
        assert c.ctx.paged_append(c.batch, 0, none[1], none[2]) is None
        assert c.ctx.paged_attention(c.batch, 0, none[0]).shape == (0, 256)
        k, v = c.ctx.paged_read(c.batch, 0, "f32")
        assert k.shape == v.shape == (sum(kv_len), 128)
        if k.shape[0]:
            assert torch.equal(k.double(), torch.cat([r[0] for r in c.rows]).view(60, 128))
    packed = g.Batch(c.ctx, None, dtype, 2, 10)
    for lens in ([0, 0], []):
        packed.set(lens)
        assert c.ctx.packed_attention(packed, 0, *none).shape == (0, 256)
    with pytest.raises(GgrError):  # what is wrong stays so
        c.ctx.paged_attention(c.batch, 1, none[0])
    with pytest.raises(ValueError):
        c.ctx.paged_attention(c.batch, 0, none[1])


def test_a_prompt_in_chunks_over_8_bit_pages():
    """The rows that 8-bit chunks are multiplied as grow with the prompt: the room for them is not made anew at every step."""
    total, step = 16384, 1024
    c = Case(16, 8, 128, "q8_head", "bf16", 64, [step], [total], seed=38)
    c.batch = g.Batch(c.ctx, c.pages, "bf16", 1, step, total // 64)
    q, free = c.q, []
    torch.empty(1 << 30, dtype=torch.uint8, device="cuda")  # (what the checks need: from torch's cache)
    for n in range(step, total + 1, step):
        c.batch.set([step], [n], c.table)
        got = c.ctx.paged_attention(c.batch, 0, q)
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
        if n in (step, 5 * step, total):
            c.kv_len, rows = [n], c.rows
            c.rows = [[x[:n] for x in rows[0]]]
            c.q = q[-40:]
            c.q_len = [40]
            out, size, reach = c.want()
            assert bool(((got[-40:].double() - out).abs() <= ref.bound(c.dtype, out, size, reach)).all())
            c.rows = rows
    assert len(set(free[1:])) <= 3, free  # 4096 rows, 8192, 16384


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("bf16", "q8_head"), ("f32", "bf16"), ("f32", "q8_head")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_layers_with_windows_of_their_own(d, kv, dtype):
    """Window and global layers of one plan: short and long texts, chunks and single tokens, cut and uncut."""
    windows = (100, 0, 33, 100, 2000)
    c = Case(8, 2, d, kv, dtype, 32, [1, 70, 3, 150], [9000, 5000, 40, 700], seed=45)
    pool, scales = ([None if x is None else x.expand(5, *x.shape[1:]).contiguous() for x in arrays] for arrays in (c.pool, c.scales))
    c.ctx = context(8, 2, d, layers=5, windows=windows)
    c.pages = g.Pages(c.ctx, c.pages.n_pages, 32, kv, *pool, *scales)
    c.batch = g.Batch(c.ctx, c.pages, dtype, 4, 224, sum(map(len, c.table)))
    c.batch.set(c.q_len, c.kv_len, c.table)
    got = [c.ctx.paged_attention(c.batch, layer, c.q) for layer in range(5)]
    for layer, window in enumerate(windows):
        c.window = window
        if layer != 3:
            c.check(got[layer])
    assert torch.equal(got[3], got[0])


def test_more_windows_than_a_plan_has_lists_for():
    ctx = context(4, 2, 64, layers=5, windows=(1, 2, 3, 4, 5))
    with pytest.raises(GgrError):
        g.Batch(ctx, None, "bf16", 1, 1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
def test_captured_steps_rotate_by_the_replayed_plan(kv, dtype):
    """Rotating append and attention of a token step in a graph, replayed at other lengths, over other pages."""
    c = Case(8, 2, 128, kv, dtype, 16, [1, 1, 1], [700, 900, 64], seed=46)
    gen = torch.Generator(device="cuda").manual_seed(47)
    q, k, v = (torch.randn(3, h * 128, generator=gen, device="cuda").to(c.dtype) for h in (8, 2, 2))
    turned, out = torch.empty_like(q), torch.empty_like(q)
    arrays = [x for x in c.pool + c.scales if x is not None]
    start = [x.clone() for x in arrays]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def step():
        c.ctx.paged_append(c.batch, 0, k, v, q=q, q_out=turned)
        c.ctx.paged_attention(c.batch, 0, turned, out=out)

    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step()
        for n, kv_len in ((3, [700, 900, 64]), (3, [12, 1, 17]), (2, [650, 800])):
            results = []
            for run in (graph.replay, step):
                for x, s in zip(arrays, start):
                    x.copy_(s)
                turned.fill_(7.0)
                out.fill_(7.0)
                c.batch.set([1] * n, kv_len, c.table[:n])
                run()
                side.synchronize()
                results.append([x.clone() for x in (turned, out, *arrays)])
            for a, b in zip(*results):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert bool((results[0][0][n:] == 7.0).all()) and bool((results[0][1][n:] == 7.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_with_strides(d, kv, dtype):
    """q as a slice of a projection's output, results into a slice of another buffer, over single tokens and chunks."""
    c = Case(8, 4, d, kv, dtype, 16, [1, 150, 20], [400, 300, 21], seed=48)
    n, dim = c.q.shape
    wide = torch.full((n, dim + 64), math.nan, dtype=c.dtype, device="cuda")
    wide[:, 32:32 + dim] = c.q
    into = torch.full((n + 1, dim + 128), 7.0, dtype=c.dtype, device="cuda")
    c.ctx.paged_attention(c.batch, 0, wide[:, 32:32 + dim], out=into[:, 64:64 + dim])
    c.check(into[:n, 64:64 + dim])
    into[:n, 64:64 + dim] = 7.0
    assert bool((into == 7.0).all())


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("bf16", "q8_head"), ("f32", "q8_head")])
def test_contexts_on_two_streams_at_once(dtype, kv):
    """Two contexts, one in a replayed graph, with launches that run beside each other: the results are those of each alone."""
    cases = [Case(8, 2, 128, kv, dtype, 16, q_len, kv_len, seed=49 + i) for i, (q_len, kv_len) in
             enumerate((([1, 200, 3], [6000, 4000, 90]), ([1, 70, 1], [9000, 3000, 1])))]
    want = [c.ctx.paged_attention(c.batch, 0, c.q).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [torch.empty_like(c.q) for c in cases]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        cases[0].ctx.paged_attention(cases[0].batch, 0, cases[0].q, out=outs[0])
        streams[0].synchronize()
        with torch.cuda.graph(graph, stream=streams[0]):
            cases[0].ctx.paged_attention(cases[0].batch, 0, cases[0].q, out=outs[0])
        graph.replay()
        streams[0].synchronize()
    first = outs[0].clone()
    cases[0].check(first)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(streams[0]):
                graph.replay()
            with torch.cuda.stream(streams[1]):
                cases[1].ctx.paged_attention(cases[1].batch, 0, cases[1].q, out=outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], first) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "q8_head"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_q_that_are_not_finite_or_large(d, kv, dtype):
    """A row of q with a NaN is a row of NaNs, and the rows beside it in its tile are right; so is a row that f16 does not hold."""
    c = Case(8, 2, d, kv, dtype, 32, [1, 150, 4], [900, 333, 60], seed=51)
    rows = c.q.view(155, 8, d)
    rows[0, 3, 7] = rows[20, 5, 0] = rows[152, 0, d - 1] = math.nan
    rows[0, 4] *= 1e5
    rows[30, 2] *= 1e5
    got = c.ctx.paged_attention(c.batch, 0, c.q).view(155, 8, d)
    spoilt = rows.isnan().any(-1)
    assert bool(got[spoilt].isnan().all())
    out, size, reach = (x.view(155, 8, d) for x in c.want())
    ok = (got.double() - out).abs() <= ref.bound(c.dtype, out, size, reach)
    assert bool(ok[~spoilt].all())
