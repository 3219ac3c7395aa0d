"""The paged-cache operators and packed-prompt attention: what is timed, in plain form and through the library's calls.

A batch is B sequences; sequence b brings `q_len[b]` new tokens, the last of the `kv_len[b]` tokens that it then has. Rows of all
sequences lie behind each other. A page holds `page` consecutive positions of one sequence, [KV head][position][element];
`table[b][j]` names the page of positions j * page and following.

Kinds of cases:
  append  RoPE of q and k, rows of k and v into their pages (bf16 pages)
  store   rows of k and v into 8-bit pages (one scale per row and KV head), and read back from there
  read    the rows of all sequences out of their pages, dense
  paged   attention of the new tokens over the pages: single tokens, chunks, or both in one batch
  packed  causal attention over whole prompts, straight from their q, k and v rows
"""
import math
import random

import numpy as np
import torch

own = False

# name: (query heads, KV heads, head_dim, adjacent-pair RoPE, theta)
SHAPES = {
    "qwen3_0p6b": (16, 8, 128, False, 1e6),
    "llama3_8b": (32, 8, 128, True, 5e5),
    "qwen3_30b_a3b": (32, 4, 128, False, 1e6),
    "gemma3_4b": (8, 4, 256, False, 1e6),
    "qwen25_14b": (40, 8, 128, False, 1e6),
    "heads_of_64": (32, 8, 64, False, 5e5),
}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # One token step of a server: every conversation appends its row, behind a prefix of its own length.
        dict(name="append_step", kind="append", shape="llama3_8b", kv="bf16", dtype="bf16", page=16, batch=24, ctx=1500, chunk=1, new="one"),
        # Several prompts come in at once, f32 rows from the projections, 8-bit pages.
        dict(name="store_prompts_q8", kind="store", shape="qwen25_14b", kv="q8", dtype="f32", page=64, batch=6, ctx=2100, chunk=2100, new="all"),
        # A short prefix out of its pages, as f32 rows.
        dict(name="read_bf16_short", kind="read", shape="qwen3_0p6b", kv="bf16", dtype="f32", page=16, batch=2, ctx=333, chunk=1, new="one"),
        # The prefixes of a batch out of 8-bit pages, to be moved or stored.
        dict(name="read_q8_long", kind="read", shape="qwen3_30b_a3b", kv="q8", dtype="bf16", page=128, batch=9, ctx=16000, chunk=1, new="one"),
        # One conversation, one token: latency.
        dict(name="decode_b1", kind="paged", shape="qwen3_0p6b", kv="bf16", dtype="bf16", page=16, batch=1, ctx=701, chunk=1, new="one", window=0),
        # A server's token step: conversations from just begun to long.
        dict(name="decode_ragged", kind="paged", shape="llama3_8b", kv="bf16", dtype="bf16", page=64, batch=48, ctx=8000, chunk=1, new="one", window=0),
        # The same on 8-bit pages with f32 rows, as the engine's projections leave them.
        dict(name="decode_q8_f32", kind="paged", shape="qwen3_30b_a3b", kv="q8", dtype="f32", page=32, batch=16, ctx=20000, chunk=1, new="one", window=0),
        # Prompts are cut into chunks that run beside the token steps of the other conversations.
        dict(name="mixed_chunks", kind="paged", shape="llama3_8b", kv="bf16", dtype="bf16", page=32, batch=12, ctx=4000, chunk=500, new="some", window=0),
        # One long prompt on 8-bit pages, a late chunk of it.
        dict(name="chunk_q8_long", kind="paged", shape="qwen25_14b", kv="q8", dtype="bf16", page=128, batch=1, ctx=16384, chunk=2048, new="chunk", window=0),
        # Chunks of three conversations on a sliding-window layer.
        dict(name="chunk_window", kind="paged", shape="gemma3_4b", kv="bf16", dtype="bf16", page=64, batch=3, ctx=6000, chunk=700, new="chunk", window=1024),
        # Short texts scored together, f32.
        dict(name="packed_short_f32", kind="packed", shape="heads_of_64", kv="bf16", dtype="f32", page=16, batch=11, ctx=280, chunk=280, new="all", window=0),
        # Long prompts of different lengths in one launch.
        dict(name="packed_long", kind="packed", shape="llama3_8b", kv="bf16", dtype="bf16", page=16, batch=3, ctx=6000, chunk=6000, new="all", window=0),
    ]


def _log_int(rng, lo, hi):
    """A whole number of lo .. hi, evenly spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    """Another case of the same kinds: one of ten patterns, with sizes from its range."""
    pattern = rng.randrange(10)
    shape, page = rng.choice([s for s in SHAPES if s != "gemma3_4b"]), rng.choice((16, 32, 64, 128, 256))
    kv, dtype = rng.choice(("bf16", "q8")), rng.choice(("bf16", "bf16", "f32"))
    hq, hkv, d = SHAPES[shape][:3]
    if pattern == 0:
        batch = _log_int(rng, 1, 64)
        return dict(kind="append", shape=shape, kv="bf16", dtype=dtype, page=page, batch=batch, ctx=_log_int(rng, 30, 3000), chunk=1, new="one")
    if pattern == 1:
        batch = _log_int(rng, 1, 12)
        ctx = _log_int(rng, 40, 2500)
        return dict(kind="append", shape=shape, kv="bf16", dtype=dtype, page=page, batch=batch, ctx=ctx, chunk=max(1, ctx // rng.choice((1, 3))), new="chunk")
    if pattern == 2:
        ctx = _log_int(rng, 20, 3000)
        return dict(kind="store", shape=shape, kv="q8", dtype=dtype, page=page, batch=_log_int(rng, 1, 10), ctx=ctx, chunk=ctx, new="all")
    if pattern == 3:
        batch = _log_int(rng, 1, 12)
        return dict(kind="read", shape=shape, kv=kv, dtype=dtype, page=page, batch=batch, ctx=_log_int(rng, 100, 60000 // batch), chunk=1, new="one")
    if pattern in (4, 5):
        batch = _log_int(rng, 1, 60)
        return dict(kind="paged", shape=shape, kv=kv, dtype=dtype, page=page, batch=batch, ctx=_log_int(rng, 50, min(20000, 400000 // batch)), chunk=1,
                    new="one", window=0)
    if pattern == 6:
        batch = _log_int(rng, 2, 14)
        ctx = _log_int(rng, 200, 5000 if dtype == "bf16" else 2000)
        return dict(kind="paged", shape=shape, kv=kv, dtype=dtype, page=page, batch=batch, ctx=ctx, chunk=_log_int(rng, 2, min(500, ctx)), new="some", window=0)
    if pattern == 7:
        batch = _log_int(rng, 1, 3)
        ctx = _log_int(rng, 100, 16000 // batch if dtype == "bf16" else 3000 // batch)
        return dict(kind="paged", shape=shape, kv=kv, dtype=dtype, page=page, batch=batch, ctx=ctx, chunk=_log_int(rng, 2, min(1500, ctx)), new="chunk", window=0)
    if pattern == 8:
        batch = _log_int(rng, 1, 5)
        ctx = _log_int(rng, 300, 6000)
        new = rng.choice(("one", "some", "chunk"))
        return dict(kind="paged", shape="gemma3_4b", kv=kv, dtype=dtype, page=page, batch=batch, ctx=ctx, chunk=1 if new == "one" else _log_int(rng, 2, min(700, ctx)),
                    new=new, window=rng.choice((0, 512, 1024)))
    batch = _log_int(rng, 1, 16)
    ctx = _log_int(rng, 30, 9000 // batch if dtype == "bf16" else 2500 // batch)
    return dict(kind="packed", shape=shape, kv="bf16", dtype=dtype, page=16, batch=batch, ctx=ctx, chunk=ctx, new="all", window=rng.choice((0, 0, 256)))


def _lengths(case):
    """(q_len, kv_len) of every sequence. They belong to the case, not to the seed: kv_len is spread from ctx / 16 to ctx."""
    r = random.Random(case["ctx"] * 131 + case["batch"] * 7 + case["chunk"])
    ctx, chunk = case["ctx"], case["chunk"]
    kv = [ctx] + [max(1, round(ctx * 16.0 ** -r.random())) for _ in range(case["batch"] - 1)]
    if case["new"] == "all":
        return kv[:], kv
    if case["new"] == "one":
        return [1] * len(kv), kv
    if case["new"] == "some":  # every third sequence has a chunk, the others a token
        return [min(n, max(1, round(chunk * (0.4 + 0.6 * r.random())))) if b % 3 == 0 else 1 for b, n in enumerate(kv)], kv
    return [min(n, chunk if b == 0 else max(1, round(chunk * (0.3 + 0.7 * r.random())))) for b, n in enumerate(kv)], kv


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    hq, hkv, d, adjacent, theta = SHAPES[case["shape"]]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    q_len, kv_len = _lengths(case)
    page, total, kind = case["page"], sum(q_len), case["kind"]
    dtype = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def index(values):
        return torch.tensor(values, dtype=torch.long, device="cuda")

    s = {"case": case, "q_len": q_len, "kv_len": kv_len}
    # keys have some channels that are larger than the others, as trained models do
    loud = 1.0 + 2.0 * (torch.rand(hkv * d, generator=gen, device="cuda") > 0.97)
    s["q"] = randn(total, hq * d).to(dtype)
    s["k"], s["v"] = (randn(total, hkv * d) * loud).to(dtype), randn(total, hkv * d).to(dtype)
    if kind == "packed":
        table = None
    else:
        used = [-(-n // page) for n in kv_len]
        n_pages = sum(used) + 3
        order = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
        at = _starts(used)
        table = [order[at[b]:at[b + 1]] for b in range(len(kv_len))]
        wide = max(used)
        s["table"] = index([row + [0] * (wide - len(row)) for row in table])
        s["pool_k"] = randn(n_pages, hkv, page, d) * loud.view(1, hkv, 1, d)
        s["pool_v"] = randn(n_pages, hkv, page, d)
        if case["kv"] == "bf16":
            s["pool_k"], s["pool_v"] = s["pool_k"].bfloat16(), s["pool_v"].bfloat16()
            s["scale_k"] = s["scale_v"] = None
        else:
            for name in ("k", "v"):
                x = s["pool_" + name]
                scale = x.abs().amax(-1) / torch.full((), 127.0, device="cuda")
                s["scale_" + name] = scale
                s["pool_" + name] = (x / scale.unsqueeze(-1)).round_().clamp_(-127, 127).to(torch.int8)
    # where the plain form finds its rows: sequence and position of every new token, and of every token
    s["seq"] = index([b for b, n in enumerate(q_len) for _ in range(n)])
    s["row"] = index([i for n in q_len for i in range(n)])
    s["pos"] = index([m - n + i for n, m in zip(q_len, kv_len) for i in range(n)])
    s["all_seq"] = index([b for b, n in enumerate(kv_len) for _ in range(n)])
    s["all_pos"] = index([p for n in kv_len for p in range(n)])
    s["first"] = index([m - n for n, m in zip(q_len, kv_len)])
    if own:
        import gguf_runner_b200 as g
        window = case.get("window", 0)
        s["ctx"] = g.AttnContext(g.AttnConfig(
            n_layers=1, n_heads=hq, n_kv_heads=hkv, head_dim=d, seq_len=8, rope_theta=theta, kv_format=g.binding.KV_BF16,
            rope_style=g.binding.ROPE_ADJACENT if adjacent else g.binding.ROPE_NEOX, swa_pattern=0, layer_windows=(window,)))
        s["pages"] = None
        if table is not None:
            s["pages"] = g.Pages(s["ctx"], n_pages, page, "bf16" if case["kv"] == "bf16" else "q8_head", k=s["pool_k"], v=s["pool_v"],
                                 k_scale=s["scale_k"], v_scale=s["scale_v"])
        s["batch"] = g.Batch(s["ctx"], s["pages"], case["dtype"], max_seqs=len(q_len), max_tokens=total,
                             max_pages=0 if table is None else sum(used))
        s["batch"].set(q_len, kv_len, table)
        if kind in ("store", "read"):
            s["out"] = [torch.empty(sum(kv_len), hkv * d, dtype=dtype, device="cuda") for _ in range(2)]
        else:
            s["out"] = torch.empty(total, hq * d, dtype=dtype, device="cuda")
    return s


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"append": _plain_append, "store": _plain_store, "read": _plain_read, "paged": _plain_paged, "packed": _plain_packed}[kind](s)
    ctx, batch, out = s["ctx"], s["batch"], s["out"]
    if kind == "append":
        ctx.paged_append(batch, 0, s["k"], s["v"], q=s["q"], q_out=out)
        return {"q": out, "k": s["pool_k"], "v": s["pool_v"]}
    if kind == "store":
        ctx.paged_append(batch, 0, s["k"], s["v"])
    if kind in ("store", "read"):
        ctx.paged_read(batch, 0, s["case"]["dtype"], k_out=out[0], v_out=out[1])
        return {"k": out[0], "v": out[1]}
    if kind == "paged":
        return ctx.paged_attention(batch, 0, s["q"], out=out)
    return ctx.packed_attention(batch, 0, s["q"], s["k"], s["v"], out=out)


# ---- plain forms ---------------------------------------------------------------------------------


def _rotate(x, pos, adjacent, theta):
    """RoPE of x [tokens][heads][d] over the whole head, angles in 64 bits."""
    d = x.shape[-1]
    power = torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d
    angle = pos.double().unsqueeze(1) * theta ** -power
    c, sn = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    x = x.float()
    if adjacent:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2)
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat((a * c - b * sn, a * sn + b * c), -1)


def _slots(s, seq, pos):
    page = s["case"]["page"]
    return s["table"][seq, pos // page], pos % page


def _plain_append(s):
    hq, hkv, d, adjacent, theta = SHAPES[s["case"]["shape"]]
    total = s["q"].shape[0]
    q = _rotate(s["q"].view(total, hq, d), s["pos"], adjacent, theta).to(s["q"].dtype)
    k = _rotate(s["k"].view(total, hkv, d), s["pos"], adjacent, theta)
    page, at = _slots(s, s["seq"], s["pos"])
    s["pool_k"][page, :, at] = k.bfloat16()
    s["pool_v"][page, :, at] = s["v"].view(total, hkv, d).bfloat16()
    return {"q": q.view(total, hq * d), "k": s["pool_k"], "v": s["pool_v"]}


def _quantise(x):
    """8-bit codes and scales of x [tokens][KV heads][d]: the steps in 32 bits, the rounding (half away from zero) in 64."""
    top = x.float().abs().amax(-1)
    n127 = torch.full_like(top, 127.0)
    some = top > 0
    factor = torch.where(some, n127 / top, torch.zeros_like(top))
    y = x.float() * factor.unsqueeze(-1)
    code = torch.sign(y) * torch.floor(y.double().abs() + 0.5).float().clamp(max=127)
    return code.to(torch.int8), torch.where(some, top / n127, torch.ones_like(top))


def _plain_store(s):
    hkv, d = SHAPES[s["case"]["shape"]][1:3]
    page, at = _slots(s, s["seq"], s["pos"])
    for name in ("k", "v"):
        code, scale = _quantise(s[name].view(-1, hkv, d))
        s["pool_" + name][page, :, at] = code
        s["scale_" + name][page, :, at] = scale
    return _plain_read(s)


def _plain_read(s):
    hkv, d = SHAPES[s["case"]["shape"]][1:3]
    page, at = _slots(s, s["all_seq"], s["all_pos"])

    def dense(pool, scale):
        x = pool[page, :, at].float()
        if scale is not None:
            x = x * scale[page, :, at].unsqueeze(-1)
        return x.to(TYPES[s["case"]["dtype"]]).view(-1, hkv * d)

    return {"k": dense(s["pool_k"], s["scale_k"]), "v": dense(s["pool_v"], s["scale_v"])}


def _attend(s, k, v, key_count):
    """Rows of the new tokens against k and v [sequence][KV head][key][d] in 32 bits; sequences and chunks padded to the longest."""
    case = s["case"]
    hq, hkv, d = SHAPES[case["shape"]][:3]
    batch, longest, total = len(s["q_len"]), max(s["q_len"]), s["q"].shape[0]
    q = torch.zeros(batch, longest, hq, d, device="cuda")
    q[s["seq"], s["row"]] = s["q"].view(total, hq, d).float()
    q = q.view(batch, longest, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, d)
    score = (q @ k.transpose(-1, -2)).view(batch, hkv, hq // hkv, longest, key_count)
    score *= 1.0 / math.sqrt(d)
    pos = (s["first"].unsqueeze(1) + torch.arange(longest, device="cuda")).unsqueeze(-1)
    key = torch.arange(key_count, device="cuda")
    hidden = key > pos
    if case["window"]:
        hidden |= key <= pos - case["window"]
    score.masked_fill_(hidden.view(batch, 1, 1, longest, key_count), -math.inf)
    score -= score.amax(-1, keepdim=True).clamp_(min=-3e38)
    score.exp_()
    total_weight = score.sum(-1, keepdim=True)
    out = (score.view(batch, hkv, -1, key_count) @ v).view(batch, hkv, hq // hkv, longest, d) / total_weight
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, longest, hq * d)
    return out[s["seq"], s["row"]].to(s["q"].dtype)


def _plain_paged(s):
    hkv, d = SHAPES[s["case"]["shape"]][1:3]
    batch, wide = s["table"].shape
    keys = wide * s["case"]["page"]

    def rows(pool, scale):
        x = pool[s["table"]].float()
        if scale is not None:
            x *= scale[s["table"]].unsqueeze(-1)
        return x.permute(0, 2, 1, 3, 4).reshape(batch, hkv, keys, d)

    return _attend(s, rows(s["pool_k"], s["scale_k"]), rows(s["pool_v"], s["scale_v"]), keys)


def _plain_packed(s):
    hkv, d = SHAPES[s["case"]["shape"]][1:3]
    batch, longest, total = len(s["q_len"]), max(s["q_len"]), s["q"].shape[0]

    def rows(x):
        padded = torch.zeros(batch, hkv, longest, d, device="cuda")
        padded[s["seq"], :, s["row"]] = x.view(total, hkv, d).float()
        return padded

    return _attend(s, rows(s["k"]), rows(s["v"]), longest)


# ---- work and exact values -----------------------------------------------------------------------


def _pairs(case):
    """(visible (token, key) pairs, keys that any new token sees), summed over the sequences."""
    pairs = keys = 0
    window = case.get("window") or 1 << 60
    for n, m in zip(*_lengths(case)):
        first = m - n
        full = min(n, max(0, window - first))  # tokens that see all keys before them
        pairs += full * first + full * (full + 1) // 2 + (n - full) * min(window, 1 << 40)
        keys += min(m, window + n - 1)
    return pairs, keys


def work(case):
    hq, hkv, d = SHAPES[case["shape"]][:3]
    q_len, kv_len = _lengths(case)
    new, total, e = sum(q_len), sum(kv_len), BYTES[case["dtype"]]
    row = hkv * (2 * d if case["kv"] == "bf16" else d + 4)  # a row of K or V in its pages
    if case["kind"] == "append":
        return {"bytes": new * d * e * (2 * hq + 2 * hkv) + 2 * new * row, "flops": 6 * new * (hq + hkv) * d}
    if case["kind"] == "store":
        return {"bytes": 2 * new * hkv * d * e + 4 * new * row + 2 * total * hkv * d * e, "flops": 8 * new * hkv * d}
    if case["kind"] == "read":
        return {"bytes": 2 * total * (row + hkv * d * e), "flops": 2 * total * hkv * d}
    pairs, keys = _pairs(case)
    kv_bytes = 2 * keys * row if case["kind"] == "paged" else 2 * new * hkv * d * e
    return {"bytes": kv_bytes + 2 * new * hq * d * e, "flops": 4 * hq * d * pairs}


def exact(case, seed):
    """What run() returns, in 64 bits: sequence by sequence, for attention one KV head at a time."""
    hq, hkv, d, adjacent, theta = SHAPES[case["shape"]]
    s = prepare(case, seed)
    q_at, kv_at = _starts(s["q_len"]), _starts(s["kv_len"])
    kind, page = case["kind"], case["page"]

    def turn(x, first):
        n, heads = x.shape[0], x.shape[1]
        z = x.double()
        out = torch.empty_like(z)
        for i in range(d // 2):
            a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + d // 2)
            angle = (torch.arange(n, dtype=torch.float64, device="cuda") + first) * math.exp(-math.log(theta) * 2 * i / d)
            c, sn = torch.cos(angle).view(n, 1), torch.sin(angle).view(n, 1)
            out[:, :, a] = z[:, :, a] * c - z[:, :, b] * sn
            out[:, :, b] = z[:, :, a] * sn + z[:, :, b] * c
        return out.view(n, heads, d)

    def grid(x):
        # the steps that the cache format defines in 32 bits, taken one by one; the value that code and scale stand for in 64
        z = x.float().cpu().numpy()
        top = np.abs(z).max(-1, keepdims=True)
        factor = np.divide(np.float32(127), top, out=np.zeros_like(top), where=top > 0)
        code = np.minimum(np.floor(np.abs(z * factor).astype(np.float64) + 0.5), 127.0) * np.sign(z)
        return torch.from_numpy(code * (top / np.float32(127)).astype(np.float64)).cuda()

    def cached(name, b):  # [key][KV head][d] of sequence b
        ids = s["table"][b, :-(-s["kv_len"][b] // page)]
        x = s["pool_" + name].index_select(0, ids).double()
        if s["scale_" + name] is not None:
            x = x * s["scale_" + name].index_select(0, ids).double().unsqueeze(-1)
        return x.transpose(1, 2).reshape(-1, hkv, d)[:s["kv_len"][b]]

    def of(name, b, heads):
        return s[name][q_at[b]:q_at[b + 1]].view(-1, heads, d)

    if kind == "append":
        q = torch.cat([turn(of("q", b, hq), s["kv_len"][b] - s["q_len"][b]).view(-1, hq * d) for b in range(len(q_at) - 1)])
        pools = {"k": s["pool_k"].double(), "v": s["pool_v"].double()}
        for b in range(len(q_at) - 1):
            first = s["kv_len"][b] - s["q_len"][b]
            rows = {"k": turn(of("k", b, hkv), first), "v": of("v", b, hkv).double()}
            at = torch.arange(first, s["kv_len"][b], device="cuda")
            for name in ("k", "v"):
                pools[name][s["table"][b, at // page], :, at % page] = rows[name]
        return {"q": q, "k": pools["k"], "v": pools["v"]}
    if kind == "store":
        return {name: torch.cat([grid(of(name, b, hkv)).view(-1, hkv * d) for b in range(len(q_at) - 1)]) for name in ("k", "v")}
    if kind == "read":
        return {name: torch.cat([cached(name, b).reshape(-1, hkv * d) for b in range(len(kv_at) - 1)]) for name in ("k", "v")}
    out = torch.empty(q_at[-1], hq, d, dtype=torch.float64, device="cuda")
    group = hq // hkv
    for b in range(len(q_at) - 1):
        k, v = (cached("k", b), cached("v", b)) if kind == "paged" else (of("k", b, hkv).double(), of("v", b, hkv).double())
        p = torch.arange(s["kv_len"][b] - s["q_len"][b], s["kv_len"][b], device="cuda").view(-1, 1)
        j = torch.arange(s["kv_len"][b], device="cuda").view(1, -1)
        seen = j <= p
        if case["window"]:
            seen &= j > p - case["window"]
        q = of("q", b, hq).double()
        for h in range(hq):
            logit = q[:, h] @ k[:, h // group].T / math.sqrt(d)
            out[q_at[b]:q_at[b + 1], h] = torch.softmax(torch.where(seen, logit, torch.full_like(logit, -math.inf)), -1) @ v[:, h // group]
    return out.view(q_at[-1], hq * d)
