"""The 4-bit KV cache and beam search, measured case by case.

Four operators: `store` (quantise keys and values into the paged 4-bit cache
and read them back), `attention` (over that cache: one token per sequence,
prompt chunks, ragged batches), `beam` (the selection over beams and
vocabulary) and `reorder` (the caches of a beam search following the selected
parents). Each has a plain form in elementary torch operations and a call of
the library (`own`); both take the same state.

The cache's pages, as include/g4cuda.h documents them: for each page and kv
head, page_size / 16 records of 16 tokens, each 17 * head_dim bytes: K codes
(8 * head_dim bytes), V codes (the same), K scales and V scales (bf16). With
G = head_dim / 64 groups of 64 dimensions a record is
  K codes  [G][key & 7][dim / 16 & 3][key >> 3][8 bytes], dim & 15 = nibble
  V codes  [G][dim / 8 & 7][key >> 1 & 3][key >> 3][key & 1][4 bytes], dim & 7 = nibble
  K scales [key][G]
  V scales [G][key >> 1 & 3][key >> 3][key & 1]
A nibble n stands for (n - 8) * scale, scale = bf16(max|x| / 7) of the group.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------
# cases

def _case(name, op, **more):
    return {"name": name, "op": op, **more}


def listed():
    return [
        # one decode step of 64 sequences: every row into its own page, 256-wide sliding-layer heads
        _case("store_step_64", "store", n=64, lo=100, hi=8704, q=1, heads=8, kv=1, hd=256, page=64, type="f32", lens=1),
        # a 512-token prefill chunk of a global layer that starts inside a page
        _case("store_chunk_512", "store", n=1, lo=1513, hi=1513, q=512, heads=8, kv=1, hd=512, page=64, type="f32",
              lens=2),
        # 16 prompts written at once, 8 kv heads of 128, bf16
        _case("store_prompts_bf16", "store", n=16, lo=4096, hi=9000, q=4096, heads=32, kv=8, hd=128, page=128,
              type="bf16", lens=3),
        # one token of one sequence on a sliding layer: the smallest call, all latency
        _case("attn_one_window", "attention", n=1, lo=777, hi=777, q=1, heads=8, kv=1, hd=256, page=64, window=512,
              type="f32", lens=4),
        # one token of one sequence at the longest context of a global layer
        _case("attn_one_131072", "attention", n=1, lo=131072, hi=131072, q=1, heads=8, kv=1, hd=512, page=64, window=0,
              type="f32", lens=5),
        # a 64-sequence serving step of a global layer, contexts of 128 to 8704 tokens
        _case("attn_serve_64", "attention", n=64, lo=128, hi=8704, q=1, heads=8, kv=1, hd=512, page=64, window=0,
              type="f32", lens=6),
        # a 32-sequence step with grouped heads in bf16
        _case("attn_serve_gqa", "attention", n=32, lo=200, hi=16384, q=1, heads=32, kv=8, hd=128, page=128, window=0,
              type="bf16", lens=7),
        # the last 512-token chunk of a 16384-token prompt on a global layer
        _case("attn_chunk_512", "attention", n=1, lo=16384, hi=16384, q=512, heads=8, kv=1, hd=512, page=64, window=0,
              type="f32", lens=8),
        # one user's search with four beams over the model's vocabulary
        _case("beam_1x4", "beam", n=1, beams=4, vocab=262144, type="f32", finished=False),
        # 16 searches of 8 beams, some hypotheses finished
        _case("beam_16x8", "beam", n=16, beams=8, vocab=262144, type="f32", finished=True),
        # the caches of one search of four beams: 12 sliding layers
        _case("reorder_1x4", "reorder", n=1, beams=4, layers=12, kv=1, hd=256, page=64, lo=437, hi=437, lens=11),
        # the caches of 16 searches of 8 beams over 15 layers that own one
        _case("reorder_16x8", "reorder", n=16, beams=8, layers=15, kv=1, hd=512, page=64, lo=200, hi=2000, lens=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def _padded(case):
    """Values that the plain form lays out at once (sequences padded to the longest)."""
    if case["op"] != "attention":
        return 0
    ctx, q = max(p + m for p, m in _spans(case)), max(m for _, m in _spans(case))
    return case["n"] * ctx * max(case["kv"] * case["hd"], q * case["heads"])


def draw(rng):
    op = rng.choice(["store", "attention", "attention", "beam", "reorder"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op in ("store", "attention"):
            kv = rng.choice([1, 1, 2, 4, 8])
            c = dict(op=op, n=_log_int(rng, 1, 64), lo=1, hi=1, q=1, kv=kv, heads=kv * rng.choice([1, 2, 4, 5, 8, 8]),
                     hd=rng.choice([64, 128, 256, 512]), page=rng.choice([16, 32, 64, 128, 256]),
                     type=rng.choice(["f32", "bf16", "f16"]), lens=rng.randrange(1 << 20))
            c["hi"] = _log_int(rng, 1, 131072)
            c["lo"] = _log_int(rng, 1, c["hi"])
            if rng.random() < 0.6:
                c["q"] = _log_int(rng, 1, 4096)
            if op == "attention":
                c["window"] = rng.choice([0, 0, 0, 512, 1000])
        elif op == "beam":
            c = dict(op=op, n=_log_int(rng, 1, 64), beams=rng.choice([1, 2, 3, 4, 5, 8, 12, 16]),
                     vocab=_log_int(rng, 1000, 262144), type=rng.choice(["f32", "bf16", "f16"]),
                     finished=rng.random() < 0.5)
        else:
            c = dict(op=op, n=_log_int(rng, 1, 32), beams=rng.choice([2, 3, 4, 5, 8, 16]), layers=_log_int(rng, 1, 35),
                     kv=rng.choice([1, 1, 2, 8]), hd=rng.choice([64, 128, 256, 512]), page=rng.choice([16, 32, 64, 128]),
                     lo=1, hi=_log_int(rng, 1, 4096), lens=rng.randrange(1 << 20))
        if _cost(c) <= most and _padded(c) <= 1 << 30:
            return c


def _spans(case):
    """(first position, tokens) of each sequence of a cache case."""
    rng = random.Random(case["lens"])
    spans = []
    for _ in range(case["n"]):
        end = _log_int(rng, case["lo"], case["hi"])
        q = case["q"] if case["n"] == 1 else rng.randint(1, case["q"])
        q = min(q, end)
        spans.append((end - q, q))
    return spans


def _lengths(case):
    rng = random.Random(case["lens"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"])]


def work(case):
    op = case["op"]
    if op in ("store", "attention"):
        spans, hd, kv, es = _spans(case), case["hd"], case["kv"], ESIZE[case["type"]]
        rows = sum(q for _, q in spans)
        if op == "store":
            # keys and values in, codes and scales out and in again, values out
            return {"bytes": rows * kv * hd * (2 * es + 2 * es + 2 * 17 / 16), "flops": rows * kv * hd * 8}
        keys = pairs = 0
        for p0, q in spans:
            w = case["window"] or p0 + q
            keys += min(p0 + q, w + q - 1)
            # position p sees min(p + 1, w) keys
            short = min(max(w - p0, 0), q)
            pairs += short * (p0 + 1) + short * (short - 1) // 2 + (q - short) * w
        return {"bytes": keys * kv * hd * 17 / 16 + 2 * rows * case["heads"] * hd * es,
                "flops": 4 * pairs * case["heads"] * hd}
    if op == "beam":
        n = case["n"] * case["beams"]
        return {"bytes": n * case["vocab"] * ESIZE[case["type"]] + 26 * n, "flops": 3 * n * case["vocab"]}
    moved = 1 - 1 / case["beams"]   # a beam that keeps its own parent copies nothing
    recs = sum(-(-(length % case["page"]) // 16) for length in _lengths(case))
    entries = sum(-(-(length + 1) // case["page"]) for length in _lengths(case))
    return {"bytes": case["beams"] * (moved * recs * case["layers"] * case["kv"] * 17 * case["hd"] * 2 + entries * 8),
            "flops": case["beams"] * entries}


# ---------------------------------------------------------------------------
# states

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _quantise(x):
    """[..., hd] -> codes + 8 (uint8) [..., G, 64] and scales [..., G]."""
    x = x.unflatten(-1, (-1, 64)).float()
    s = (x.abs().amax(-1) / 7).to(torch.bfloat16)
    return torch.round(x / s.float().unsqueeze(-1)).clamp(-7, 7).add(8).to(torch.uint8), s


def _records(k, v):
    """Keys and values [..., 16, hd] as the cache's records [..., 17 * hd] (uint8)."""
    lead = k.shape[:-2]
    z = len(lead)

    def order(t, *dims):
        return t.permute(*range(z), *[z + d for d in dims]).contiguous()

    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    g = kc.shape[-2]
    kc = order(kc.reshape(*lead, 2, 8, g, 4, 8, 2), 2, 1, 3, 0, 4, 5)
    vc = order(vc.reshape(*lead, 2, 4, 2, g, 8, 4, 2), 3, 4, 1, 0, 2, 5, 6)
    vs = order(vs.reshape(*lead, 2, 4, 2, g), 3, 1, 0, 2)
    parts = [(c[..., 0] | (c[..., 1] << 4)).reshape(*lead, -1) for c in (kc, vc)]
    parts += [s.reshape(*lead, -1).contiguous().view(torch.uint8) for s in (ks, vs)]
    return torch.cat(parts, -1)


def _pool(pages, kv, recs, hd, g):
    """A pool of pages that hold RMS-normalised keys and values, [pages][kv][recs][17 * hd]."""
    out = torch.empty((pages, kv, recs, 17 * hd), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (kv * recs * 16 * hd))
    for i in range(0, pages, step):
        m = min(step, pages - i)
        k, v = _randn((2, m, kv, recs, 16, hd), g)
        k /= k.square().mean(-1, keepdim=True).sqrt()
        v /= v.square().mean(-1, keepdim=True).sqrt()
        out[i:i + m] = _records(k, v)
    return out


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("store", "attention"):
        spans, kv, hd, page = _spans(case), case["kv"], case["hd"], case["page"]
        rows = sum(q for _, q in spans)
        s["offsets"] = _ints(np.cumsum([0] + [q for _, q in spans]).tolist())
        s["start"] = _ints([p for p, _ in spans])
        held = [-(-(p + q) // page) for p, q in spans]
        total, stride = sum(held), max(held)
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["n"], stride), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, m in enumerate(held):
            table[i, :m] = ids[at:at + m]
            at += m
        s["table"], s["rows"] = table, rows
        dtype = TYPES[case["type"]]
        if op == "store":
            s["pool"] = torch.zeros((total, kv, page // 16, 17 * hd), dtype=torch.uint8, device="cuda")
            # keys and values as they come out of one projection: rows of q | k | v
            heads = case["heads"]
            qkv = _randn((rows, heads + 2 * kv, hd), g, dtype)
            s["k"], s["v"] = qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        else:
            s["pool"] = _pool(total, kv, page // 16, hd, g)
            s["q"] = _randn((rows, case["heads"], hd), g, dtype)
            s["scale"] = 2.0 / math.sqrt(hd)
    elif op == "beam":
        n, w, v = case["n"], case["beams"], case["vocab"]
        x = 4 * torch.randn((n * w, v), generator=g, device="cuda")
        s["logits"] = (30 * torch.tanh(x / 30)).to(TYPES[case["type"]])
        s["scores"] = -20 * torch.rand((n, w), generator=g, device="cuda")
        s["finished"] = (torch.rand((n, w), generator=g, device="cuda") < (0.25 if case["finished"] else 0)).to(
            torch.uint8)
        s["eos"] = 1
    else:
        n, w, layers, page = case["n"], case["beams"], case["layers"], case["page"]
        lengths = _lengths(case)
        s["lengths"] = _ints(lengths)
        stride = max(length // page for length in lengths) + 2
        # each beam's own pages: what it may write from here on, and a spare one; the full pages are shared
        full = [length // page for length in lengths]
        total = sum(full) + n * w * 3
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        table = torch.full((n, w, stride), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, m in enumerate(full):
            table[i, :, :m] = ids[at:at + m]
            at += m
            table[i, :, m:m + 2] = ids[at:at + 2 * w].reshape(w, 2)
            at += 2 * w
        s["table"], s["spare"] = table.reshape(n * w, stride), ids[at:at + n * w].clone()
        s["parents"] = torch.randint(0, w, (n, w), generator=g, device="cuda", dtype=torch.int32)
        s["pool"] = torch.randint(0, 256, (layers, total, case["kv"], page // 16, 17 * case["hd"]), generator=g,
                                  device="cuda", dtype=torch.uint8)
    return s


# ---------------------------------------------------------------------------
# plain forms

def _values(rec):
    """Records [..., 17 * hd] as keys and values [..., 16, hd] in fp32."""
    lead, hd = rec.shape[:-1], rec.shape[-1] // 17
    z, g = len(lead), hd // 64

    def order(t, *dims):
        return t.permute(*range(z), *[z + d for d in dims])

    def codes(b):
        return torch.stack((b & 15, b >> 4), -1).float() - 8

    ks = rec[..., 16 * hd:16 * hd + 32 * g].contiguous().view(torch.bfloat16).float().reshape(*lead, 16, g, 1)
    vs = rec[..., 16 * hd + 32 * g:].contiguous().view(torch.bfloat16).float().reshape(*lead, g, 4, 2, 2)
    vs = order(vs, 2, 1, 3, 0).reshape(*lead, 16, g, 1)
    k = order(codes(rec[..., :8 * hd].reshape(*lead, g, 8, 4, 2, 8)), 3, 1, 0, 2, 4, 5).reshape(*lead, 16, g, 64)
    v = order(codes(rec[..., 8 * hd:16 * hd].reshape(*lead, g, 8, 4, 2, 2, 4)), 3, 2, 4, 0, 1, 5, 6)
    v = v.reshape(*lead, 16, g, 64)
    return (k * ks).flatten(-2), (v * vs).flatten(-2)


def _stored(x):
    """[..., hd] -> the values that its 4-bit codes stand for, quantised in 64 bits (codes next to a border)."""
    y = x.unflatten(-1, (-1, 64)).double()
    s = (y.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).double()
    c = torch.where(s > 0, torch.round(y / s), 0).clamp(-7, 7)
    return c, s


def _where(s):
    """Sequence and position of every row."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    return row, seq, s["start"].long()[seq] + row - s["offsets"].long()[seq]


def _plain_store(s):
    case = s["case"]
    page, hd = case["page"], case["hd"]
    g = hd // 64
    _, seq, pos = _where(s)
    at = s["table"].long()[seq, pos // page]
    rec, tok = pos % page // 16, pos % 16
    lead = (s["rows"], case["kv"])
    (kc, ks), (vc, vs) = _stored(s["k"]), _stored(s["v"])
    out = []
    pool = s["pool"]
    for c, sc, key in ((kc, ks, True), (vc, vs, False)):
        n = (c + 8).to(torch.uint8).reshape(*lead, -1, 2)
        b = n[..., 0] | (n[..., 1] << 4)                   # [rows, kv, hd / 2]
        i = torch.arange(hd // 2, device="cuda")
        if key:
            where = i // 32 * 512 + (tok[:, None] & 7) * 64 + i // 8 % 4 * 16 + (tok[:, None] >> 3) * 8 + i % 8
            j = torch.arange(g, device="cuda")
            sat = 8 * hd + tok[:, None] * g + j
        else:
            where = (8 * hd + i // 32 * 512 + i // 4 % 8 * 64 + (tok[:, None] >> 1 & 3) * 16 + (tok[:, None] >> 3) * 8
                     + (tok[:, None] & 1) * 4 + i % 4)
            j = torch.arange(g, device="cuda")
            sat = (8 * hd + 16 * g + j * 16 + (tok[:, None] >> 1 & 3) * 4 + (tok[:, None] >> 3) * 2
                   + (tok[:, None] & 1))
        h = torch.arange(case["kv"], device="cuda")
        pool[at[:, None, None], h[None, :, None], rec[:, None, None], where[:, None, :]] = b
        half = pool.view(torch.bfloat16)
        half[at[:, None, None], h[None, :, None], rec[:, None, None], sat[:, None, :]] = (
            sc.squeeze(-1).to(torch.bfloat16))
        out.append((c * sc).flatten(-2).to(TYPES[case["type"]]))
    return out


def _plain_attention(s):
    case = s["case"]
    n, kv, hd, heads = case["n"], case["kv"], case["hd"], case["heads"]
    row, seq, pos = _where(s)
    local = row - s["offsets"].long()[seq]
    rec = s["pool"][s["table"].long().clamp(min=0)]       # [n, stride, kv, recs, 17 hd]
    k, v = _values(rec.permute(0, 2, 1, 3, 4))             # [n, kv, stride, recs, 16, hd]
    k, v = k.flatten(2, 4), v.flatten(2, 4)
    most = int(case["q"]) if n > 1 else s["rows"]
    q = torch.zeros((n, most, heads, hd), device="cuda")
    q[seq, local] = s["q"].float()
    at = torch.full((n, most), -1, dtype=torch.long, device="cuda")
    at[seq, local] = pos
    q = q.reshape(n, most, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    sc = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    j = torch.arange(k.shape[2], device="cuda")
    see = j <= at[..., None]
    if case["window"]:
        see &= j > at[..., None] - case["window"]
    see = see.repeat_interleave(heads // kv, 1)[:, None]   # [n, 1, most * group, keys]
    sc = torch.where(see, sc, -torch.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m > -torch.inf, m, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    o = o.reshape(n, kv, most, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, most, heads, hd)
    return o[seq, local].to(s["q"].dtype)


def _plain_beam(s):
    n, w, vocab = s["case"]["n"], s["case"]["beams"], s["case"]["vocab"]
    x = s["logits"].double().reshape(n, w, vocab)          # 64 bits: candidates of two beams may lie close
    m = x.amax(-1, keepdim=True)
    cand = s["scores"].double()[..., None] + (x - m - (x - m).exp().sum(-1, keepdim=True).log())
    done = s["finished"].bool()[..., None]
    stay = torch.where(torch.arange(vocab, device="cuda") == s["eos"], s["scores"].double()[..., None], -torch.inf)
    cand = torch.where(done, stay, cand).reshape(n, -1)
    best, at = torch.sort(cand, dim=-1, descending=True, stable=True)
    best, at = best[:, :w], at[:, :w]
    parents, tokens = at // vocab, at % vocab
    ended = s["finished"].gather(1, parents) | (tokens == s["eos"]).to(torch.uint8)
    return best.float(), parents.int(), tokens.int(), ended


def _plain_reorder(s):
    case = s["case"]
    n, w, page = case["n"], case["beams"], case["page"]
    i = torch.arange(n * w, device="cuda")
    parent = (s["parents"].long() + torch.arange(n, device="cuda")[:, None] * w).flatten()
    full = (s["lengths"].long() // page).repeat_interleave(w)
    left = (s["lengths"].long() % page).repeat_interleave(w)
    table, spare = s["table"], s["spare"]
    j = torch.arange(table.shape[1], device="cuda")
    out = torch.where(j < full[:, None], table[parent], table)
    moved = (parent != i) & (left > 0)
    out = torch.where(moved[:, None] & (j == full[:, None]), spare[:, None], out)
    own_page = table[i, full]
    spare_out = torch.where(moved, own_page, spare)
    src, dst = table[parent, full].long(), spare.long()
    rec = torch.arange(page // 16, device="cuda")
    take = moved[:, None] & (rec < (left[:, None] + 15) // 16)
    pool = s["pool"]
    pool[:, dst] = torch.where(take[None, :, None, :, None], pool[:, src], pool[:, dst])
    return out, spare_out, pool.view(torch.int32)


PLAIN = {"store": _plain_store, "attention": _plain_attention, "beam": _plain_beam, "reorder": _plain_reorder}


# ---------------------------------------------------------------------------
# the library's calls

def _g4():
    if "g4cuda" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "gemma4.c_b200"))
    import g4cuda
    return g4cuda


def _handle(s, make):
    """The descriptors and the workspace that a program keeps beside its cache."""
    if "handle" not in s:
        s["handle"] = make(_g4())
    return s["handle"]


def _cache(g4, s, pool=None):
    case = s["case"]
    pool = s["pool"] if pool is None else pool
    return g4.Kv4Cache(pool.data_ptr(), pool.shape[0], case["page"], case["kv"], case["hd"])


def _own_store(s):
    def make(g4):
        return (g4, _cache(g4, s),
                g4.Kv4Batch(s["case"]["n"], s["rows"], s["offsets"].data_ptr(), s["start"].data_ptr(),
                            s["table"].data_ptr(), s["table"].shape[1]),
                getattr(g4, "TYPE_" + s["case"]["type"].upper()))
    g4, cache, batch, kind = _handle(s, make)
    k, v = s["k"], s["v"]
    ko = torch.empty(k.shape, dtype=k.dtype, device="cuda")
    vo = torch.empty(v.shape, dtype=v.dtype, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    g4.kv4_write(cache, batch, kind, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), st)
    g4.kv4_read(cache, batch, kind, ko.data_ptr(), ko.stride(0), vo.data_ptr(), vo.stride(0), st)
    return [ko, vo]


def _own_attention(s):
    def make(g4):
        cache = _cache(g4, s)
        batch = g4.Kv4Batch(s["case"]["n"], s["rows"], s["offsets"].data_ptr(), s["start"].data_ptr(),
                            s["table"].data_ptr(), s["table"].shape[1])
        kind = getattr(g4, "TYPE_" + s["case"]["type"].upper())
        size = g4.kv4_attention_workspace(cache, batch, kind, s["case"]["heads"])
        return g4, cache, batch, kind, torch.empty(size, dtype=torch.uint8, device="cuda")
    g4, cache, batch, kind, ws = _handle(s, make)
    q = s["q"]
    out = torch.empty_like(q)
    g4.kv4_attention(cache, batch, kind, s["case"]["heads"], q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0),
                     s["scale"], s["case"]["window"], ws.data_ptr(), ws.numel(),
                     torch.cuda.current_stream().cuda_stream)
    return out


def _own_beam(s):
    case = s["case"]
    n, w, vocab = case["n"], case["beams"], case["vocab"]

    def make(g4):
        return (g4, getattr(g4, "TYPE_" + case["type"].upper()),
                torch.empty(g4.beam_workspace(n, w, vocab), dtype=torch.uint8, device="cuda"))
    g4, kind, ws = _handle(s, make)
    scores = torch.empty((n, w), dtype=torch.float32, device="cuda")
    ints = torch.empty((2, n, w), dtype=torch.int32, device="cuda")
    ended = torch.empty((n, w), dtype=torch.uint8, device="cuda")
    x = s["logits"]
    g4.beam_select(n, w, vocab, kind, x.data_ptr(), x.stride(0), s["scores"].data_ptr(), s["finished"].data_ptr(),
                   s["eos"], scores.data_ptr(), ints[0].data_ptr(), ints[1].data_ptr(), ended.data_ptr(),
                   ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    return scores, ints[0], ints[1], ended


def _own_reorder(s):
    def make(g4):
        return g4, g4.kv4_caches([_cache(g4, s, p) for p in s["pool"]])
    g4, caches = _handle(s, make)
    table, spare = torch.empty_like(s["table"]), torch.empty_like(s["spare"])
    g4.kv4_reorder(caches, s["case"]["n"], s["case"]["beams"], s["parents"].data_ptr(), s["lengths"].data_ptr(),
                   s["table"].data_ptr(), table.data_ptr(), table.shape[1], s["spare"].data_ptr(), spare.data_ptr(),
                   torch.cuda.current_stream().cuda_stream)
    return table, spare, s["pool"].view(torch.int32)


OWN = {"store": _own_store, "attention": _own_attention, "beam": _own_beam, "reorder": _own_reorder}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits

def _bf16_round(x):
    """fp64 array (non-negative) -> the nearest bf16 values, ties to even significands."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 256), e - 8)


def _exact_stored(x):
    x = x.double().cpu().numpy()
    y = x.reshape(*x.shape[:-1], -1, 64)
    s = _bf16_round(np.max(np.abs(y), -1, keepdims=True) / 7)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.clip(np.rint(y / s), -7, 7), 0)
    return (c * s).reshape(x.shape)


def _map(hd):
    """Where token t, dimension d of a record lies: byte and shift of the K and V nibbles, bf16 index of the scales."""
    t, d = np.meshgrid(np.arange(16), np.arange(hd), indexing="ij")
    grp, low = d // 64, d % 64
    kb = grp * 512 + (t % 8) * 64 + (low // 16) * 16 + (t // 8) * 8 + (low % 16) // 2
    vb = 8 * hd + grp * 512 + (low // 8) * 64 + (t % 8 // 2) * 16 + (t // 8) * 8 + (t % 2) * 4 + (low % 8) // 2
    ki = 8 * hd + t * (hd // 64) + grp
    vi = 8 * hd + hd // 4 + grp * 16 + (t % 8 // 2) * 4 + (t // 8) * 2 + t % 2
    return [torch.from_numpy(a).cuda() for a in (kb, vb, ki, vi, 4 * (d % 2))]


def _exact_attention(s):
    case = s["case"]
    kv, hd, heads, window = case["kv"], case["hd"], case["heads"], case["window"]
    kb, vb, ki, vi, shift = _map(hd)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    offsets, starts = s["offsets"].tolist(), s["start"].tolist()
    for b in range(case["n"]):
        r0, r1, p0 = offsets[b], offsets[b + 1], starts[b]
        end = p0 + r1 - r0
        pages = s["table"][b, :-(-end // case["page"])].long()
        for h in range(kv):
            rec = s["pool"][pages, h].reshape(-1, 17 * hd)
            half = rec.view(torch.bfloat16)
            k, v = (((rec[:, byte] >> shift & 15).double() - 8) * half[:, idx].double() for byte, idx in
                    ((kb, ki), (vb, vi)))
            k, v = k.reshape(-1, hd)[:end], v.reshape(-1, hd)[:end]
            per = heads // kv
            for r in range(r0, r1, 128):
                e = min(r1, r + 128)
                q = s["q"][r:e, h * per:(h + 1) * per].double()
                sc = torch.einsum("rhd,kd->rhk", q, k) * s["scale"]
                pos = torch.arange(p0 + r - r0, p0 + e - r0, device="cuda")[:, None, None]
                j = torch.arange(end, device="cuda")
                hidden = (j > pos) | ((j <= pos - window) if window else False)
                out[r:e, h * per:(h + 1) * per] = torch.einsum(
                    "rhk,kd->rhd", torch.softmax(sc.masked_fill(hidden, -torch.inf), -1), v)
    return out


def _exact_beam(s):
    n, w, vocab = s["case"]["n"], s["case"]["beams"], s["case"]["vocab"]
    scores, parents, tokens, ended = [], [], [], []
    for i in range(n):
        cand = torch.log_softmax(s["logits"][i * w:(i + 1) * w].double(), -1) + s["scores"][i].double()[:, None]
        for b in range(w):
            if s["finished"][i, b]:
                cand[b] = -torch.inf
                cand[b, s["eos"]] = s["scores"][i, b].double()
        cand = cand.flatten()
        for _ in range(w):
            best = cand.max()
            at = int(torch.nonzero(cand == best)[0])
            scores.append(best.item())
            parents.append(at // vocab)
            tokens.append(at % vocab)
            ended.append(int(s["finished"][i, at // vocab]) | int(at % vocab == s["eos"]))
            cand[at] = torch.nan
            cand = torch.nan_to_num(cand, nan=-torch.inf, neginf=-torch.inf)
    return (np.array(scores).reshape(n, w), np.array(parents, np.int32).reshape(n, w),
            np.array(tokens, np.int32).reshape(n, w), np.array(ended, np.uint8).reshape(n, w))


def exact(case, seed):
    if case["op"] == "reorder":
        return None                                        # whole numbers and copies: nothing is computed
    s = prepare(case, seed)
    if case["op"] == "store":
        return [_exact_stored(s["k"]), _exact_stored(s["v"])]
    if case["op"] == "attention":
        w = work(case)
        return _exact_attention(s) if w["flops"] < 2e12 else None
    return _exact_beam(s)
