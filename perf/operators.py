"""Measured cases of the 4-bit key/value cache operators and of token scoring.

Operators (C ABI, include/midgecuda.h):
  append    mg_kv4_append, mg_kv4_read  per-head RMSNorm of queries and keys, rotary position, keys and
                                        values stored in 4 bits in a paged cache (and read back)
  attn      mg_kv4_attn                 attention of new queries over that cache: single tokens, a few
                                        tokens, prompt chunks; sinks, sliding window, grouped heads
  logprobs  mg_logprobs                 log probabilities of given tokens, entropy, top alternatives

The cache: pages of `page` positions; a page holds, for each key/value head, page / 32 tiles of 32
positions.  A tile of head_dim D has G = D / 32 groups of 32 dimensions and 32 D + 64 G bytes:
  [0, 16 D)             keys, e2m1 codes, low nibble = even dimension
  [16 D, 32 D)          values, the same
  [32 D, 32 D + 32 G)   the keys' scales, one e5m2 byte per position and group
  [.. + 32 G)           the values' scales
in the order of the lanes of a tensor-core fragment (_K_SHAPE and the others below give the order of
the axes).  A value is its code times its scale.
"""
import math
import random

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MIDPOINTS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
ACT = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
# (query heads, key/value heads, head_dim): the shapes of the configurations, one with a head of
# keys for each query head, one with groups that are no power of two, one with a single key head
HEADS = ((64, 8, 64), (32, 4, 128), (4, 2, 64), (16, 16, 64), (40, 8, 128), (16, 1, 128))
VOCABS = (201088, 151936, 32000, 1024)


def listed():
    return [
        # one decode step of the benchmark: 8 sequences, a token each, around position 4096
        dict(name="append-decode-8", op="append", type="f32", heads=64, kv=8, dim=64, seqs=8, tokens=8, first=4096, norm=False, page=64),
        # the benchmark's prompt of 4096 tokens
        dict(name="append-prompt-4096", op="append", type="f32", heads=64, kv=8, dim=64, seqs=1, tokens=4096, first=0, norm=False, page=64),
        # chunks of five prompts of a model with query and key norms, uneven lengths
        dict(name="append-norm-8191", op="append", type="bf16", heads=32, kv=4, dim=128, seqs=5, tokens=8191, first=777, norm=True, page=128),
        # a single chat, just begun: latency
        dict(name="attn-first-tokens", op="attn", type="f32", heads=64, kv=8, dim=64, seqs=1, q=1, shortest=129, longest=129, window=0, sinks=True, page=64),
        # one decode step of the benchmark: 8 sequences at 4096
        dict(name="attn-decode-8x4096", op="attn", type="f32", heads=64, kv=8, dim=64, seqs=8, q=1, shortest=4096, longest=4096, window=0, sinks=True, page=64),
        # the same model's sliding layers, many sequences of all lengths
        dict(name="attn-decode-window", op="attn", type="f32", heads=64, kv=8, dim=64, seqs=128, q=1, shortest=1, longest=8192, window=128, sinks=True, page=32),
        # a full server: 64 sequences, 1 to 32768 tokens each
        dict(name="attn-decode-64-long", op="attn", type="bf16", heads=32, kv=4, dim=128, seqs=64, q=1, shortest=1, longest=32768, window=0, sinks=False, page=128),
        # checking five drafted tokens of each of 16 sequences
        dict(name="attn-verify-5", op="attn", type="f16", heads=64, kv=8, dim=64, seqs=16, q=5, shortest=1500, longest=9001, window=0, sinks=True, page=64),
        # the benchmark's prompt of 4096 tokens, all of it new
        dict(name="attn-prompt-4096", op="attn", type="f32", heads=64, kv=8, dim=64, seqs=1, q=4096, shortest=4096, longest=4096, window=0, sinks=True, page=64),
        # chunks of three long prompts, the cache filled before them
        dict(name="attn-chunk-1009", op="attn", type="bf16", heads=32, kv=4, dim=128, seqs=3, q=1009, shortest=5003, longest=16384, window=0, sinks=False, page=128),
        # the logits of one decode step: the chosen token, five alternatives
        dict(name="logprobs-decode-8", op="logprobs", type="f32", vocab=201088, rows=8, ids=1, top=5),
        # scoring a prompt of 2048 tokens with twenty alternatives at each
        dict(name="logprobs-prompt-2047", op="logprobs", type="bf16", vocab=151936, rows=2047, ids=1, top=20),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def draw(rng):
    op = rng.choice(("append", "attn", "attn", "logprobs"))
    kind = rng.choice(("f32", "f32", "f16", "bf16"))
    if op == "logprobs":
        vocab = rng.choice(VOCABS + (_log(rng, 100, 200000),))
        rows = _log(rng, 1, min(4096, 300_000_000 // vocab))
        return dict(op=op, type=kind, vocab=vocab, rows=rows, ids=rng.choice((1, 1, 4)), top=rng.choice((0, 1, 5, 20, 32)))
    heads, kv, dim = rng.choice(HEADS)
    page = rng.choice((32, 64, 128, 256))
    if op == "append":
        tokens = _log(rng, 1, 8000)
        return dict(op=op, type=kind, heads=heads, kv=kv, dim=dim, seqs=_log(rng, 1, min(tokens, 64)), tokens=tokens, first=_log(rng, 1, 16000), norm=rng.random() < 0.5, page=page)
    window = rng.choice((0, 0, 0, 128, _log(rng, 1, 4000)))
    form = rng.choice(("single", "single", "few", "chunk"))
    q = 1 if form == "single" else rng.randint(2, 16) if form == "few" else _log(rng, 17, 2048)
    seqs = _log(rng, 1, 64) if form != "chunk" else rng.randint(1, 4)
    room = 1_000_000 // seqs if form == "single" else 400_000 // seqs if form == "few" else min(16384, 4_000_000_000 // (seqs * q * heads * 4))
    longest = max(q, _log(rng, 1, min(32768, room)))
    return dict(op=op, type=kind, heads=heads, kv=kv, dim=dim, seqs=seqs, q=q, shortest=max(q, longest // rng.choice((1, 2, 10))) if form != "single" else rng.choice((1, longest)),
                longest=longest, window=window, sinks=rng.random() < 0.5, page=page)


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """The sequences' lengths: spread evenly from the shortest to the longest, in a fixed shuffled order."""
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    v = [b if n == 1 else a + (b - a) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(v)
    return v


def _spread(case):
    """append: the tokens of each sequence, uneven, and the position of its first."""
    n, t = case["seqs"], case["tokens"]
    w = [1 + (7 * i) % 5 for i in range(n)]
    c = [1 + (t - n) * x // sum(w) for x in w]
    c[0] += t - sum(c)
    return c, [case["first"] + (0 if n == 1 else 13 * i) for i in range(n)]


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _tile_bytes(dim):
    return 32 * dim + 2 * dim


# order of the axes in a tile: u = half of the tile, n j = pair and member (p = 16 u + 2 n + j);
# t = quarter of the dimensions; t i = quad and member (p = 16 u + 4 t + i, i = c + 2 s), g = eighth of the dimensions
def _k_from(b, dim):  # [..., 16 dim] bytes -> [..., 32 positions, dim / 2 bytes]
    e = b.shape[:-1]
    n = len(e)
    x = b.view(*e, 2, 8, 4, 2, 8).permute(*range(n), n, n + 1, n + 3, n + 2, n + 4) if dim == 64 else b.view(*e, 2, 2, 8, 4, 16).permute(*range(n), n, n + 2, n + 1, n + 3, n + 4)
    return x.reshape(*e, 32, dim // 2)


def _v_from(b, dim):
    e = b.shape[:-1]
    n = len(e)
    x = b.view(*e, 2, 8, 4, 4, 4).permute(*range(n), n, n + 2, n + 3, n + 1, n + 4) if dim == 64 else b.view(*e, 2, 2, 8, 4, 2, 8).permute(*range(n), n, n + 3, n + 4, n + 1, n + 2, n + 5)
    return x.reshape(*e, 32, dim // 2)


def _ks_from(b, dim):  # [..., 32 G] -> [..., 32, G]
    e, n = b.shape[:-1], b.dim() - 1
    return b.view(*e, 8, dim // 32, 2, 2).permute(*range(n), n + 2, n, n + 3, n + 1).reshape(*e, 32, dim // 32)


def _vs_from(b, dim):
    e, n = b.shape[:-1], b.dim() - 1
    return b.view(*e, 4, dim // 32, 2, 4).permute(*range(n), n + 2, n, n + 3, n + 1).reshape(*e, 32, dim // 32)


def _k_to(x, dim):  # the inverse orders
    e, n = x.shape[:-2], x.dim() - 2
    y = x.view(*e, 2, 8, 2, 4, 8).permute(*range(n), n, n + 1, n + 3, n + 2, n + 4) if dim == 64 else x.view(*e, 2, 8, 2, 4, 16).permute(*range(n), n, n + 2, n + 1, n + 3, n + 4)
    return y.reshape(*e, 16 * dim)


def _v_to(x, dim):
    e, n = x.shape[:-2], x.dim() - 2
    y = x.view(*e, 2, 4, 4, 8, 4).permute(*range(n), n, n + 3, n + 1, n + 2, n + 4) if dim == 64 else x.view(*e, 2, 4, 2, 2, 8, 8).permute(*range(n), n, n + 3, n + 4, n + 1, n + 2, n + 5)
    return y.reshape(*e, 16 * dim)


def _ks_to(x, dim):
    e, n = x.shape[:-2], x.dim() - 2
    return x.view(*e, 2, 8, 2, dim // 32).permute(*range(n), n + 1, n + 3, n, n + 2).reshape(*e, dim)


def _vs_to(x, dim):
    e, n = x.shape[:-2], x.dim() - 2
    return x.view(*e, 2, 4, 4, dim // 32).permute(*range(n), n + 1, n + 3, n, n + 2).reshape(*e, dim)


def _e5m2(b):
    return (b.to(torch.int16) << 8).view(torch.float16).float()


def _quantise(x):
    """[..., dim] -> bytes [..., dim / 2] and scale bytes [..., dim / 32]: the scale is the least e5m2 >= largest / 6, from 2^-14 to
    10240; the code is the nearest e2m1, ties to the even code."""
    x = x.unflatten(-1, (-1, 32)).float()
    top = x.abs().amax(-1)
    steps = torch.arange(4, 4 * 28 + 2, device=x.device, dtype=torch.uint8)  # e5m2 bytes from 2^-14 to 10240, ascending
    at = torch.searchsorted(_e5m2(steps) * 6, top).clamp(max=len(steps) - 1)
    sb = torch.where(top == 0, 0, steps[at])
    s = _e5m2(sb).unsqueeze(-1)
    a = x.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, m in enumerate(MIDPOINTS):
        code += (a > m * s) if i % 2 == 0 else (a >= m * s) & (s > 0)
    code |= (x < 0).to(torch.uint8) << 3
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, sb


def _values(b, sb):
    """bytes [..., dim / 2] and scale bytes [..., dim / 32] -> 32-bit values [..., dim]"""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=b.device)
    pair = torch.stack((lut.repeat(16), lut.repeat_interleave(16)), 1)  # of a byte: even dimension, odd dimension
    v = pair[b.int()].flatten(-2)
    return (v.unflatten(-1, (-1, 32)) * _e5m2(sb).unsqueeze(-1)).flatten(-2)


def _rope(rows, dim):
    """YaRN tables of the benchmark's model (theta 150000, factor 32, 4096 positions originally), 32 bits"""
    half = dim // 2
    inv = 150000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    at = [dim * math.log(4096 / (beta * 2 * math.pi)) / (2 * math.log(150000.0)) for beta in (32.0, 1.0)]
    keep = 1 - ((torch.arange(half, dtype=torch.float64, device="cuda") - at[0]) / (at[1] - at[0])).clamp(0, 1)
    inv = inv / 32 * (1 - keep) + inv * keep
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    m = 0.1 * math.log(32.0) + 1
    return (a.cos() * m).float(), (a.sin() * m).float()


def _table(g, lengths, page):
    """Pages in random order: [sequences, most pages] and how many there are"""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need), generator=g, device="cuda").int()
    table, at = torch.zeros(len(need), max(1, max(need)), dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = ACT[case["type"]][0]
    s = dict(case=case)
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # a flat floor with a few clear winners of a random height, and a share of the tokens banned
        x = torch.empty(rows, vocab, dtype=dt, device="cuda")
        for r in range(0, rows, 256):
            part = _normal(g, min(256, rows - r), vocab) * 2
            hot = torch.randint(vocab, (part.shape[0], 8), generator=g, device="cuda")
            part.scatter_add_(1, hot, 12 * torch.rand(hot.shape, generator=g, device="cuda"))
            part[:, vocab // 2:vocab // 2 + vocab // 100] = -math.inf
            x[r:r + 256] = part
            del part
        ids = torch.randint(vocab // 2, (rows, case["ids"]), generator=g, device="cuda", dtype=torch.int32)
        ids[:, 0] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, x.argmax(1).int(), ids[:, 0])
        s |= dict(logits=x, ids=ids, lp=torch.empty(rows, case["ids"], device="cuda"), entropy=torch.empty(rows, device="cuda"),
                  top_ids=torch.empty(rows, case["top"], dtype=torch.int32, device="cuda"), top_lp=torch.empty(rows, case["top"], device="cuda"))
        return s
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    if case["op"] == "append":
        count, first = _spread(case)
        lengths = [a + b for a, b in zip(count, first)]
        table, pages = _table(g, lengths, page)
        s["pool"] = torch.zeros(pages, kv, page // 32, _tile_bytes(dim), dtype=torch.uint8, device="cuda")
        x = _normal(g, case["tokens"], (heads + 2 * kv) * dim)  # a fused projection's rows: queries, keys, values
        x[:, heads * dim:(heads + kv) * dim].view(-1, kv, dim)[:, :, 3::29] *= 6  # keys have channels of their own size
        s["qkv"] = x.to(dt)
        s["q_norm"], s["k_norm"] = 1 + 0.1 * _normal(g, dim), 1 + 0.1 * _normal(g, dim)
        s["cos"], s["sin"] = _rope(max(lengths), dim)
        s["seq"] = torch.tensor([i for i, n in enumerate(count) for _ in range(n)], dtype=torch.int32, device="cuda")
        s["pos"] = torch.tensor([first[i] + j for i, n in enumerate(count) for j in range(n)], dtype=torch.int32, device="cuda")
        s["q_out"] = torch.empty(case["tokens"], heads * dim, dtype=dt, device="cuda")
        s["k_out"], s["v_out"] = (torch.empty(case["tokens"], kv * dim, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    else:
        lengths = _lengths(case)
        table, pages = _table(g, lengths, page)
        pool = torch.empty(pages, kv, page // 32, _tile_bytes(dim), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 25) // (kv * page * dim))
        for a in range(0, pages, step):
            n = min(step, pages - a)
            k, v = _normal(g, n, kv, page // 32, 32, dim), _normal(g, n, kv, page // 32, 32, dim)
            k[..., 3::29] *= 4
            (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
            pool[a:a + n] = torch.cat((_k_to(kc, dim), _v_to(vc, dim), _ks_to(ks, dim), _vs_to(vs, dim)), -1)
        s["pool"] = pool
        n = case["seqs"] * case["q"]
        s["q"] = (1.2 * _normal(g, n, heads * dim)).to(dt)
        s["out"] = torch.empty(n, heads * dim, dtype=dt, device="cuda")
        s["sinks"] = _normal(g, heads) if case["sinks"] else None
        s["q_start"] = torch.arange(case["seqs"] + 1, dtype=torch.int32, device="cuda") * case["q"]
        s["kv_len"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["longest"] = max(lengths)
        s["scale"] = dim ** -0.5
    s["table"] = table
    return s


# ------------------------------------------------------------- plain forms


def _plain_append(s):
    c = s["case"]
    heads, kv, dim, page, n = c["heads"], c["kv"], c["dim"], c["page"], c["tokens"]
    dt = ACT[c["type"]][0]
    x = s["qkv"].float().view(n, heads + 2 * kv, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if c["norm"]:
        q = q * (1 / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * s["q_norm"]
        k = k * (1 / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * s["k_norm"]
    pos = s["pos"].long()
    co, si = s["cos"][pos, None], s["sin"][pos, None]
    turn = lambda y: torch.cat((y[..., :dim // 2] * co - y[..., dim // 2:] * si, y[..., dim // 2:] * co + y[..., :dim // 2] * si), -1)  # noqa: E731
    q, k = turn(q), turn(k)
    # the places of the tokens' bytes: the tile's numbers put through the tile's order
    at = torch.arange(_tile_bytes(dim), device="cuda")
    order = [_k_from(at[:16 * dim], dim), _v_from(at[16 * dim:32 * dim], dim), _ks_from(at[32 * dim:33 * dim], dim), _vs_from(at[33 * dim:], dim)]
    tile = (s["table"][s["seq"].long(), pos // page].long() * kv)[:, None] + torch.arange(kv, device="cuda")
    base = (tile * (page // 32) + (pos % page // 32)[:, None]) * _tile_bytes(dim)
    flat = s["pool"].view(-1)
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    idx = [base[..., None] + o[pos % 32][:, None] for o in order]
    flat[idx[0]], flat[idx[1]], flat[idx[2]], flat[idx[3]] = kc, vc, ks, vs
    k, v = _values(flat[idx[0]], flat[idx[2]]), _values(flat[idx[1]], flat[idx[3]])
    return {"q": q.reshape(n, -1).to(dt), "k": k.reshape(n, -1).bfloat16(), "v": v.reshape(n, -1).bfloat16()}


def _plain_attn(s):
    c = s["case"]
    heads, kv, dim, n, b = c["heads"], c["kv"], c["dim"], c["q"], c["seqs"]
    tiles = s["pool"][s["table"].long()].transpose(1, 2).flatten(2, 3)  # [b, kv, tiles, bytes]
    q = s["q"].float().view(b, n, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, dim)
    k = _values(_k_from(tiles[..., :16 * dim], dim), _ks_from(tiles[..., 32 * dim:33 * dim], dim)).flatten(2, 3)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"])
    del k
    at = torch.arange(score.shape[-1], device="cuda")
    pos = (s["kv_len"][:, None] - n + torch.arange(n, device="cuda"))[..., None]  # [b, n, 1]
    hidden = (at > pos) | (at <= pos - c["window"]) if c["window"] else at > pos
    score.view(b, kv, n, heads // kv, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    if c["sinks"]:
        sink = s["sinks"].view(kv, 1, heads // kv).expand(kv, n, heads // kv).reshape(kv, -1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0, m)
    p = score.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    if c["sinks"]:
        total = total + (sink - m).exp()
    v = _values(_v_from(tiles[..., 16 * dim:32 * dim], dim), _vs_from(tiles[..., 33 * dim:], dim)).flatten(2, 3)
    out = torch.matmul(p, v)
    out = torch.where(total > 0, out / total, 0)
    return out.view(b, kv, n, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(b * n, -1).to(ACT[c["type"]][0])


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    z = total.log()
    lp = d.gather(1, s["ids"].long()) - z
    entropy = (z - torch.where(e > 0, e * d, 0).sum(-1, keepdim=True) / total)[:, 0]
    del e
    best = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
    return {"lp": lp, "entropy": entropy, "top_ids": best.int(), "top_lp": d.gather(1, best) - z}


# --------------------------------------------------- the framework's calls


def _cache(s):
    from midge_b200 import abi

    c = s["case"]
    return abi.MgKv4(n_kv_heads=c["kv"], head_dim=c["dim"], page_size=c["page"], n_pages=s["pool"].shape[0], pages=s["pool"].data_ptr(),
                     table=s["table"].data_ptr(), ld_table=s["table"].shape[1], n_seqs=s["table"].shape[0])


def _calls(s):
    """The argument lists of the calls on this state's buffers, laid out once as a serving loop keeps them"""
    import ctypes as C

    from midge_b200 import abi

    c, lib = s["case"], abi.lib
    act = ACT[c["type"]][1]
    ptr = lambda t: C.c_void_p(t.data_ptr() if t is not None and t.numel() else None)  # noqa: E731
    if c["op"] == "logprobs":
        work = torch.zeros(max(1, abi.check_size(lib.mg_logprobs_work(c["vocab"], c["rows"], c["top"]))), dtype=torch.uint8, device="cuda")
        s["keep"] = work
        return [(lib.mg_logprobs, (act, ptr(s["logits"]), c["vocab"], c["vocab"], c["rows"], ptr(s["ids"]), c["ids"], c["top"], ptr(s["lp"]), ptr(s["entropy"]),
                                   ptr(s["top_ids"]), ptr(s["top_lp"]), ptr(work), work.numel()))]
    cache = _cache(s)
    ref = C.byref(cache)
    if c["op"] == "append":
        heads, kv, dim, n = c["heads"], c["kv"], c["dim"], c["tokens"]
        ld, size = s["qkv"].shape[1], s["qkv"].element_size()
        q, k, v = (C.c_void_p(s["qkv"].data_ptr() + size * dim * h) for h in (0, heads, heads + kv))
        s["keep"] = cache
        return [(lib.mg_kv4_append, (ref, act, n, heads, q, ld, k, ld, v, ld, ptr(s["q_norm"] if c["norm"] else None), ptr(s["k_norm"] if c["norm"] else None), 1e-6,
                                     ptr(s["cos"]), ptr(s["sin"]), s["cos"].shape[0], ptr(s["seq"]), ptr(s["pos"]), ptr(s["q_out"]), heads * dim)),
                (lib.mg_kv4_read, (ref, ACT["bf16"][1], n, ptr(s["seq"]), ptr(s["pos"]), ptr(s["k_out"]), kv * dim, ptr(s["v_out"]), kv * dim))]
    work = torch.zeros(max(1, abi.check_size(lib.mg_kv4_attn_work(ref, c["heads"], c["q"], s["longest"]))), dtype=torch.uint8, device="cuda")
    s["keep"] = (cache, work)
    ld = s["q"].shape[1]
    return [(lib.mg_kv4_attn, (ref, act, c["heads"], ptr(s["q"]), ld, ptr(s["q_start"]), ptr(s["kv_len"]), c["q"], s["longest"], s["scale"], c["window"],
                               ptr(s["sinks"]), ptr(s["out"]), ld, ptr(work), work.numel()))]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _plain_append, "attn": _plain_attn, "logprobs": _plain_logprobs}[op](s)
    calls = s.get("calls")
    if calls is None:
        calls = s["calls"] = _calls(s)
    stream = torch.cuda.current_stream().cuda_stream
    for f, args in calls:
        if f(*args, stream):
            from midge_b200 import abi

            raise RuntimeError(abi.lib.mg_last_error().decode())
    if op == "append":
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if op == "attn":
        return s["out"]
    return {"lp": s["lp"], "entropy": s["entropy"], "top_ids": s["top_ids"], "top_lp": s["top_lp"]}


# -------------------------------------------------------- the bare minimum


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (8 * case["ids"] + 8 * case["top"] + 4), "flops": 5 * n}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    entry = kv * 2 * (dim // 2 + dim // 32)  # bytes of one cached position
    if case["op"] == "append":
        n = case["tokens"]
        # rows in, queries out, codes out and in again, 16-bit values out; each position's rotation
        moved = (2 * heads + 2 * kv) * dim * size + 2 * entry + 2 * kv * dim * 2 + 8 + dim * 4
        return {"bytes": n * moved, "flops": n * ((heads + kv) * dim * (8 if case["norm"] else 3) + 4 * kv * dim)}
    seen = pairs = 0
    q, w = case["q"], case["window"]
    for n in _lengths(case):
        seen += n if not w else min(n, w + q - 1)
        a = n - q  # the first query's position
        pairs += sum(min(w, p + 1) for p in range(a, n)) if w else q * (a + 1) + q * (q - 1) // 2
    return {"bytes": seen * entry + 2 * case["seqs"] * q * heads * dim * size, "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------- in 64 bits


def _places(pos, dim, keys):
    """Byte within the tile, and shift in it, of each dimension's code, and the byte of its scale, for positions [n]: from the format's description"""
    p, d = (pos % 32)[:, None], torch.arange(dim, device=pos.device)[None]
    u, groups = p // 16, dim // 32
    if keys:
        n, j = p % 16 // 2, p % 2
        lane = n * 4 + d // (dim // 4)
        code = u * 512 + lane * 16 + j * 8 + d % 16 // 2 if dim == 64 else u * 1024 + j * 512 + lane * 16 + d % 32 // 2
        return code, d % 2 * 4, 32 * dim + (n * groups + d // 32) * 4 + u * 2 + j
    t, i = p % 16 // 4, p % 4
    lane = d // (dim // 8) * 4 + t
    code = u * 512 + lane * 16 + i * 4 + d % 8 // 2 if dim == 64 else u * 1024 + i % 2 * 512 + lane * 16 + i // 2 * 8 + d % 16 // 2
    return 16 * dim + code, d % 2 * 4, 33 * dim + ((t * groups + d // 32) * 2 + u) * 4 + i


def _stored(s, seq, length, head, keys):
    """Positions 0 .. length - 1 of one sequence and head, in 64 bits"""
    c = s["case"]
    dim, page = c["dim"], c["page"]
    pos = torch.arange(length, device="cuda")
    code, shift, scale = _places(pos, dim, keys)
    row = s["pool"].view(-1, page // 32, _tile_bytes(dim))
    tile = (s["table"][seq, pos // page].long() * c["kv"] + head, pos % page // 32)
    bits = row[tile[0][:, None], tile[1][:, None], code].int() >> shift
    exponent, fraction = bits >> 1 & 3, (bits & 1).double()
    v = torch.where(exponent == 0, fraction / 2, (1 + fraction / 2) * 2.0 ** (exponent - 1).double()) * (1 - 2.0 * (bits >> 3 & 1))
    sb = row[tile[0][:, None], tile[1][:, None], scale].int()
    e, f = sb >> 2, (sb & 3).double() / 4
    return v * torch.where(e == 0, f * 2.0 ** -14, (1 + f) * 2.0 ** (e - 15).double())


def _exact_four_bits(x):
    """The values that 4 bits keep of x [n, heads, dim], by the rule's definition"""
    n, h, dim = x.shape
    x = x.view(n, h, dim // 32, 32)
    all_scales = torch.tensor([m * 2.0 ** e for e in range(-14, 14) for m in (1, 1.25, 1.5, 1.75)][:-2], dtype=torch.float64, device="cuda")
    need = x.abs().amax(-1)
    least = torch.where(all_scales * 6 >= need[..., None], all_scales, math.inf).amin(-1).clamp(max=10240.0)[..., None]
    r = (x.abs() / least).clamp(max=6)
    # nearest: halves below 2, wholes below 4, doubles above; round() takes ties to the even step, which is the even code
    r = torch.where(r <= 2, (r * 2).round() / 2, torch.where(r <= 4, r.round(), (r / 2).round() * 2))
    return (torch.where(need[..., None] > 0, r * least, 0) * x.sign()).view(n, h * dim)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        out = {"lp": [], "entropy": [], "top_ids": [], "top_lp": []}
        for r in range(0, case["rows"], 64):
            x = s["logits"][r:r + 64].double()
            z = torch.logsumexp(x, -1, keepdim=True)
            l = x - z
            out["lp"].append(l.gather(1, s["ids"][r:r + 64].long()))
            out["entropy"].append(-(l.exp() * l.clamp(min=-1e30)).sum(-1))
            # the top ones: by value, then by index
            left, ids = x.clone(), []
            for _ in range(case["top"]):
                best = left.amax(-1, keepdim=True)
                i = torch.where(left == best, torch.arange(x.shape[1], device="cuda"), x.shape[1]).amin(-1, keepdim=True)
                ids.append(i)
                left.scatter_(1, i, -math.inf)
            i = torch.cat(ids, 1) if ids else torch.zeros(x.shape[0], 0, dtype=torch.long, device="cuda")
            out["top_ids"].append(i.int())
            out["top_lp"].append(l.gather(1, i))
        return {k: torch.cat(v) for k, v in out.items()}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if case["op"] == "append":
        n, half = case["tokens"], dim // 2
        x = s["qkv"].double()
        pos = s["pos"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[pos]

        def moved(y, weight):
            y = y.reshape(n, -1, dim)
            if case["norm"]:
                y = y / (y.pow(2).sum(-1, keepdim=True) / dim + 1e-6).sqrt() * weight.double()
            z = torch.complex(y[..., :half], y[..., half:]) * turn[:, None]
            return torch.cat((z.real, z.imag), -1)

        q = moved(x[:, :heads * dim], s["q_norm"])
        k = moved(x[:, heads * dim:(heads + kv) * dim], s["k_norm"])
        v = x[:, (heads + kv) * dim:].reshape(n, kv, dim)
        return {"q": q.reshape(n, -1), "k": _exact_four_bits(k), "v": _exact_four_bits(v)}
    n, group = case["q"], heads // kv
    out = torch.zeros(case["seqs"], n, heads, dim, dtype=torch.float64, device="cuda")
    for b, length in enumerate(_lengths(case)):
        pos = length - n + torch.arange(n, device="cuda")
        for h in range(kv):
            k, v = _stored(s, b, length, h, True), _stored(s, b, length, h, False)
            for a in range(0, n, 1024):  # some queries at a time
                p = pos[a:a + 1024, None, None]
                q = s["q"].view(case["seqs"], n, kv, group, dim)[b, a:a + 1024, h].double()
                score = torch.einsum("ngd,ld->ngl", q, k) * s["scale"]
                at = torch.arange(length, device="cuda")
                seen = (at <= p) & ((at > p - case["window"]) if case["window"] else torch.ones_like(at, dtype=torch.bool))
                score = torch.where(seen, score, -math.inf)
                if case["sinks"]:
                    sink = s["sinks"].double().view(kv, group)[h].expand(score.shape[0], group)[..., None]
                    w = torch.softmax(torch.cat((score, sink), -1), -1)[..., :-1]
                else:
                    w = torch.softmax(score, -1)
                out[b, a:a + 1024, h * group:(h + 1) * group] = torch.einsum("ngl,ld->ngd", w, v)
    return out.view(case["seqs"] * n, -1)
