"""Score a text with a 4-bit paged key/value cache.

Runs a converted model through the library's kernel-level entry points, the
way a host with its own scheduler would (several sequences share one pool of
pages; a step takes the next tokens of each): embedding rows, norms and
projections, mg_kv4_append (query/key norms, rotation, 4-bit store),
mg_kv4_attn over the pages, the router and the experts, the output logits,
and mg_logprobs.  It prints what the model says of every token of the text --
log probability, entropy, the best alternatives -- which is also how one sees
what the smaller cache costs: with --f16 the same text goes through the
engine and its f16 cache (engine/midge.c:267-273 of the reference) as well.

    python -m midge_b200.kv4_score <model_dir> --ids 12,7,99,4 [--top 5] [--page 64] [--f16]
"""
from __future__ import annotations

import argparse
import ctypes as C

import numpy as np

from . import abi
from .container import DT_CODES, ModelDir, spec_fields

STEP = 16  # tokens of a step: what one mg_moe_ffn call takes


def rope_tables(f: dict, n: int):
    """cos and sin [n, head_dim / 2] with YaRN, in double and rounded once:
    the arithmetic of engine/midge.c:141-176."""
    hd = f["head_dim"]
    half = hd // 2
    i = np.arange(half, dtype=np.float64)
    theta = float(np.float32(f["rope_theta"]))
    inv, m = 1.0 / theta ** (2 * i / hd), 1.0
    if f["yarn"]:
        orig = f["yarn_orig_ctx"]
        low, high = (hd * np.log(orig / (b * 2 * np.pi)) / (2 * np.log(theta))
                     for b in (f["yarn_beta_fast"], f["yarn_beta_slow"]))
        if f["yarn_truncate"]:
            low, high = np.floor(low), np.ceil(high)
        low, high = max(low, 0.0), min(high, hd - 1.0)
        if high == low:
            high = low + 0.001
        keep = 1.0 - np.clip((i - low) / (high - low), 0.0, 1.0)
        inv = inv / f["yarn_factor"] * (1.0 - keep) + inv * keep
        m = 0.1 * np.log(f["yarn_factor"]) + 1.0
    a = np.arange(n, dtype=np.float64)[:, None] * inv
    return (np.cos(a) * m).astype(np.float32), (np.sin(a) * m).astype(np.float32)


class Kv4Model:
    """A model's weights on the GPU and, per layer, a 4-bit cache of `seqs`
    sequences of up to `ctx` tokens whose pages come from one free list."""

    def __init__(self, path: str, ctx: int, seqs: int = 1, page: int = 64):
        import torch

        self.torch = torch
        md = ModelDir(path)
        try:
            self.f = f = spec_fields(md.spec)
            self.w = {n: (DT_CODES[dt], rows, cols, self._up(d), None if s is None else self._up(s))
                      for n, dt, rows, cols, d, s in md.tensors()}
            self.layout = abi.MgExpertLayout()
            abi.check(abi.lib.mg_expert_layout_init(C.byref(self.layout), DT_CODES[md.expert_dt], f["hidden"], f["ffn"],
                                                    f["n_experts"]))
            self.experts = self._up(md.expert_blob())
        finally:
            md.close()
        self.ctx, self.page = ctx, page
        self.cos, self.sin = (torch.from_numpy(x).cuda() for x in rope_tables(f, ctx))
        per = -(-ctx // page)
        size = abi.check_size(abi.lib.mg_kv4_page_bytes(f["n_kv_heads"], f["head_dim"], page))
        self.table = torch.zeros(seqs, per, dtype=torch.int32, device="cuda")
        self.free = list(range(seqs * per))
        self.len = [0] * seqs
        # a pool per layer; the layers share the page table
        self.pool = torch.empty(f["n_layers"], seqs * per, size, dtype=torch.uint8, device="cuda")
        self.cache = [abi.MgKv4(n_kv_heads=f["n_kv_heads"], head_dim=f["head_dim"], page_size=page, n_seqs=seqs,
                                n_pages=seqs * per, pages=self.pool[i].data_ptr(), table=self.table.data_ptr(),
                                ld_table=per) for i in range(f["n_layers"])]
        need = abi.check_size(abi.lib.mg_kv4_attn_work(C.byref(self.cache[0]), f["n_heads"], STEP, ctx))
        self.work = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def _up(self, a):
        return self.torch.from_numpy(np.array(a)).cuda()

    def _vec(self, name):
        return self.w[name][3].data_ptr()

    def _gemv(self, name, x, y, bias=None, accumulate=0, col=0):
        dt, rows, cols, d, s = self.w[name]
        abi.check(abi.lib.mg_gemv(dt, abi.MG_SCALE_F16, d.data_ptr(), None if s is None else s.data_ptr(), rows, cols,
                                  x.data_ptr(), x.shape[1], x.shape[0], None if bias is None else self._vec(bias),
                                  accumulate, y.data_ptr() + 4 * col, y.shape[1], self.stream))

    def _norm(self, x, w):
        out = self.torch.empty_like(x)
        abi.check(abi.lib.mg_rmsnorm(x.data_ptr(), self._vec(w), out.data_ptr(), x.shape[1], x.shape[0],
                                     self.f["norm_eps"], self.stream))
        return out

    def step(self, tokens):
        """tokens: {sequence: its next token ids}, STEP in all at most.
        Returns the logits [tokens, vocab] (device), sequences ascending."""
        torch, f, lib = self.torch, self.f, abi.lib
        self.stream = torch.cuda.current_stream().cuda_stream
        seqs = sorted(tokens)
        ids = [t for s in seqs for t in tokens[s]]
        n, H, hd, nh, nkv = len(ids), f["hidden"], f["head_dim"], f["n_heads"], f["n_kv_heads"]
        if not 1 <= n <= STEP or any(not 0 <= t < f["vocab"] for t in ids):
            raise ValueError(f"a step takes 1 to {STEP} tokens of the vocabulary")
        for s in seqs:
            if not 0 <= s < len(self.len) or self.len[s] + len(tokens[s]) > self.ctx:
                raise ValueError(f"sequence {s}: no such sequence, or its context is full")
        for s in seqs:  # pages for the new positions
            for p in range(-(-self.len[s] // self.page), -(-(self.len[s] + len(tokens[s])) // self.page)):
                self.table[s, p] = self.free.pop()

        def dev(v):
            return torch.tensor(v, dtype=torch.int32, device="cuda")

        count = [len(tokens.get(s, ())) for s in range(len(self.len))]
        pos = dev([self.len[s] + j for s in seqs for j in range(len(tokens[s]))])
        seq = dev([s for s in seqs for _ in tokens[s]])
        for s in seqs:
            self.len[s] += len(tokens[s])
        q_start, kv_len = dev(np.concatenate([[0], np.cumsum(count)]).tolist()), dev(self.len)

        dt, rows, cols, d, sc = self.w["embed"]
        idd, x = dev(ids), torch.empty(n, H, device="cuda")
        abi.check(lib.mg_dequant_rows(dt, abi.MG_SCALE_F16, d.data_ptr(), None if sc is None else sc.data_ptr(), rows,
                                      cols, idd.data_ptr(), n, x.data_ptr(), self.stream))
        width = (nh + 2 * nkv) * hd
        qkv, att = torch.empty(n, width, device="cuda"), torch.empty(n, nh * hd, device="cuda")
        logits = torch.empty(n, f["n_experts"], device="cuda")
        sel = torch.empty(n, f["top_k"], dtype=torch.int32, device="cuda")
        wts = torch.empty(n, f["top_k"], device="cuda")
        h = torch.empty(n * f["top_k"] * f["ffn"], device="cuda")
        for i in range(f["n_layers"]):
            p, c = f"L{i}.", C.byref(self.cache[i])
            xb = self._norm(x, p + "attn.norm")
            for name, col in (("q", 0), ("k", nh * hd), ("v", (nh + nkv) * hd)):
                self._gemv(p + "attn." + name, xb, qkv, p + f"attn.{name}_b", col=col)
            at = qkv.data_ptr()
            qn, kn = (self._vec(p + "attn.q_norm"), self._vec(p + "attn.k_norm")) if f["qk_norm"] else (None, None)
            # the queries are turned in place: q_out is q
            abi.check(lib.mg_kv4_append(c, abi.MG_ACT_F32, n, nh, at, width, at + 4 * nh * hd, width,
                                        at + 4 * (nh + nkv) * hd, width, qn, kn, f["norm_eps"], self.cos.data_ptr(),
                                        self.sin.data_ptr(), self.ctx, seq.data_ptr(), pos.data_ptr(), at, width,
                                        self.stream))
            window = f["sliding_window"] if f["layer_sliding"][i] else 0
            abi.check(lib.mg_kv4_attn(c, abi.MG_ACT_F32, nh, at, width, q_start.data_ptr(), kv_len.data_ptr(),
                                      max(count), max(self.len), f["attn_scale"], window,
                                      self._vec(p + "attn.sinks") if f["sinks"] else None, att.data_ptr(), nh * hd,
                                      self.work.data_ptr(), self.work.numel(), self.stream))
            self._gemv(p + "attn.o", att, x, p + "attn.o_b", accumulate=1)
            xb = self._norm(x, p + "mlp.norm")
            abi.check(lib.mg_router_topk(xb.data_ptr(), n, self._vec(p + "router.w"), self._vec(p + "router.b"),
                                         f["n_experts"], H, f["top_k"], f["router_norm"], 1, logits.data_ptr(),
                                         sel.data_ptr(), wts.data_ptr(), self.stream))
            abi.check(lib.mg_moe_ffn(C.byref(self.layout), self.experts.data_ptr(), i, f["n_experts"], xb.data_ptr(), n,
                                     f["top_k"], sel.data_ptr(), wts.data_ptr(), f["act_plain"], f["alpha"], f["limit"],
                                     h.data_ptr(), x.data_ptr(), self.stream))
        out = torch.empty(n, f["vocab"], device="cuda")
        self._gemv("lm_head", self._norm(x, "final_norm"), out)
        abi.check(lib.mg_kv4_attn_status(self.work.data_ptr(), self.work.numel(), self.stream))
        return out


def logprobs(logits, ids, top: int):
    """mg_logprobs of device rows: (log probability of ids[i] in row i, entropy,
    alternatives, their log probabilities) as numpy arrays."""
    import torch

    n, V = logits.shape
    idd = torch.tensor(np.asarray(ids).reshape(n, 1), dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(n, 1, device="cuda"), torch.empty(n, device="cuda")
    ai, al = torch.empty(n, top, dtype=torch.int32, device="cuda"), torch.empty(n, top, device="cuda")
    work = torch.zeros(abi.check_size(abi.lib.mg_logprobs_work(V, n, top)), dtype=torch.uint8, device="cuda")
    abi.check(abi.lib.mg_logprobs(abi.MG_ACT_F32, logits.data_ptr(), V, V, n, idd.data_ptr(), 1, top, lp.data_ptr(),
                                  ent.data_ptr(), ai.data_ptr() if top else None, al.data_ptr() if top else None,
                                  work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream))
    return lp[:, 0].cpu().numpy(), ent.cpu().numpy(), ai.cpu().numpy(), al.cpu().numpy()


def score(model: Kv4Model, ids, seq: int = 0, top: int = 5, step: int = STEP):
    """What the model says of ids[1:], each from the tokens before it: arrays
    of log probability, entropy, alternatives and theirs, one row a token."""
    # step looks at all but the last, which mg_logprobs would take for "no token": probability 1
    if len(ids) < 2 or any(not 0 <= t < model.f["vocab"] for t in ids):
        raise ValueError("two tokens of the vocabulary at least")
    parts = []
    for a in range(0, len(ids) - 1, step):
        t = list(ids[a:min(a + step, len(ids) - 1)])
        parts.append(logprobs(model.step({seq: t}), ids[a + 1:a + 1 + len(t)], top))
    return tuple(np.concatenate(x) for x in zip(*parts))


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("model")
    ap.add_argument("--ids", required=True, help="token ids, comma separated")
    ap.add_argument("--top", type=int, default=5)
    ap.add_argument("--page", type=int, default=64)
    ap.add_argument("--f16", action="store_true", help="also with the engine's f16 cache")
    a = ap.parse_args()
    ids = [int(t) for t in a.ids.split(",")]
    if len(ids) < 2:
        ap.error("two tokens at least")
    lp, ent, ai, al = score(Kv4Model(a.model, len(ids), page=a.page), ids, top=a.top)
    for i, t in enumerate(ids[1:]):
        print("%6d  lp %9.4f  entropy %7.4f  %s" % (t, lp[i], ent[i], " ".join("%d:%.3f" % x for x in zip(ai[i], al[i]))))
    print("mean log probability, 4-bit cache: %.5f" % lp.mean())
    if a.f16:
        import torch

        m = abi.Model.from_dir(a.model, ctx=len(ids))
        rows = torch.from_numpy(m.forward_batch(0, ids[:-1], logits_mode=2)).cuda()
        print("mean log probability, f16 cache:   %.5f" % logprobs(rows, ids[1:], 0)[0].mean())
        m.close()


if __name__ == "__main__":
    main()
