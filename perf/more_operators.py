"""The operators for decoding many sequences at once, over the cases a server of
them meets: rotary positions of rows, appending keys and values to a paged cache
of 8-bit blocks, attention over that cache, and the log probabilities of tokens.

  listed()              the named cases
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   inputs and buffers on the GPU
  run(state)            one pass, its outputs: the library's entry points where
                        own is true, elementary torch operations otherwise
  work(case)            bytes and operations a pass cannot do without
  exact(case, seed)     the outputs in 64 bits, written apart from run()

A layer's cache: pages of `page` tokens; a block is 16 tokens of one KV head, K
as [16][head_dim] and V as [head_dim][16] e4m3 codes, with a power of two as
scale for each of the two; pages are [KV heads][page / 16] blocks.  A call's
rows row_start[s] .. row_start[s + 1] - 1 continue the lengths[s] tokens of
sequence s, which lie in the pages that row s of the page table names.

Queries, keys and values are N(0, 1) rows, as projections of normed
activations are; logits have the spread of a language model's.
"""
from __future__ import annotations

import ctypes
import importlib
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
BLOCK = 16
INF = math.inf
E4M3 = torch.float8_e4m3fn
MOST = 448.0  # the largest e4m3 value
LEAST_SCALE = 2.0 ** -100


# ---- the cases ----------------------------------------------------------------
def listed():
    return [
        # one decoded token's q and k heads: the smallest call, all latency
        {"name": "rope_1_row", "op": "rope", "rows": 1, "heads": 40, "hd": 128, "rot": 128, "inter": 0, "yarn": 0,
         "top": 4096},
        # a prompt's rows of a model that rotates half of each head, context scaled by four
        {"name": "rope_2048_part_scaled", "op": "rope", "rows": 2048, "heads": 40, "hd": 128, "rot": 64, "inter": 1,
         "yarn": 4, "top": 131072},
        # one sequence's next token
        {"name": "append_1", "op": "append", "seqs": 1, "low": 1000, "high": 1000, "new_low": 1, "new_high": 1,
         "page": 64, "heads": 32, "kv": 8, "hd": 128, "rot": 128, "inter": 0, "yarn": 0, "norm": 1},
        # a decode step of a busy server
        {"name": "append_64", "op": "append", "seqs": 64, "low": 20, "high": 600, "new_low": 1, "new_high": 1,
         "page": 32, "heads": 32, "kv": 8, "hd": 128, "rot": 128, "inter": 0, "yarn": 0, "norm": 1},
        # new prompts of odd lengths, some behind a shared beginning that is cached already
        {"name": "append_prompts", "op": "append", "seqs": 5, "low": 0, "high": 300, "new_low": 101, "new_high": 701,
         "page": 64, "heads": 32, "kv": 8, "hd": 128, "rot": 128, "inter": 0, "yarn": 4, "norm": 1},
        # one sequence's next token: latency
        {"name": "attend_1_at_1000", "op": "attend", "seqs": 1, "low": 1000, "high": 1000, "new_low": 1, "new_high": 1,
         "page": 64, "heads": 32, "kv": 8, "hd": 128, "sw": 0},
        # one long document, a model with four KV heads
        {"name": "attend_1_at_60001", "op": "attend", "seqs": 1, "low": 60001, "high": 60001, "new_low": 1,
         "new_high": 1, "page": 64, "heads": 32, "kv": 4, "hd": 128, "sw": 0},
        # a decode step of a busy server, conversations of every length
        {"name": "attend_64_ragged", "op": "attend", "seqs": 64, "low": 100, "high": 8000, "new_low": 1,
         "new_high": 1, "page": 32, "heads": 32, "kv": 8, "hd": 128, "sw": 0},
        # chunks of prompts behind cached tokens
        {"name": "attend_prompts", "op": "attend", "seqs": 4, "low": 500, "high": 4000, "new_low": 300,
         "new_high": 700, "page": 64, "heads": 32, "kv": 8, "hd": 128, "sw": 0},
        # the answer to one decoded token, five alternatives
        {"name": "logprobs_1_top5", "op": "logprobs", "rows": 1, "vocab": 151936, "top": 5},
        # a batch's decoded tokens, twenty alternatives
        {"name": "logprobs_64_top20", "op": "logprobs", "rows": 64, "vocab": 151936, "top": 20},
        # a scored prompt over a 32000-word vocabulary
        {"name": "logprobs_1999", "op": "logprobs", "rows": 1999, "vocab": 32000, "top": 0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 8, 128), (32, 8, 128), (32, 4, 128), (64, 8, 128), (32, 1, 128), (16, 16, 64), (32, 8, 64), (8, 2, 256),
         (12, 4, 128)]


def draw(rng):
    op = rng.choice(["rope"] * 2 + ["append"] * 3 + ["attend"] * 4 + ["logprobs"] * 3)
    if op == "rope":
        hd, rows = rng.choice([64, 80, 96, 128, 128, 256]), _log(rng, 1, 2048)
        return {"op": op, "rows": rows, "heads": rng.randint(1, 10240 // max(64, hd)), "hd": hd,
                "rot": 2 * rng.choice([hd // 2, hd // 2, hd // 4, rng.randint(1, hd // 2)]), "inter": rng.choice([0, 1]),
                "yarn": rng.choice([0, 0, 4, 8]), "top": _log(rng, 100, 1000000)}
    if op == "logprobs":
        rows = _log(rng, 1, 2000)
        return {"op": op, "rows": rows, "vocab": min(_log(rng, 300, 256000), 64000000 // rows),
                "top": rng.choice([0, 1, 5, 20, rng.randint(1, 32)])}
    h, kv, hd = rng.choice(HEADS)
    seqs, page = _log(rng, 1, 100), rng.choice([16, 32, 64, 128])
    case = {"op": op, "seqs": seqs, "page": page, "heads": h, "kv": kv, "hd": hd}
    if rng.random() < 0.6:
        case |= {"new_low": 1, "new_high": 1}
    else:
        most = max(1, 1500 // seqs)
        case |= {"new_low": rng.randint(0, most) // 2, "new_high": most}
    if op == "append":
        low = rng.choice([0, 0, rng.randint(1, 300)])
        return case | {"low": low, "high": low + rng.randint(0, 300), "rot": rng.choice([hd, hd, hd // 2]),
                       "inter": rng.choice([0, 0, 1]), "yarn": rng.choice([0, 0, 4]), "norm": rng.choice([1, 1, 0, -1])}
    most = min(32768, 64 * 4096 * 8 * 128 // (seqs * kv * hd))
    if case["new_high"] > 1:
        most = max(1, min(most, 10 ** 10 // (seqs * case["new_high"] * h * hd) - case["new_high"]))
    high = _log(rng, 1, most)
    return case | {"low": rng.randint(0, high), "high": high, "sw": rng.choice([0, 0, 0, 512, 1024])}


def _sequences(case):
    """Every sequence's tokens in the cache before the call, and its new rows."""
    r = random.Random(case["seqs"] * 1000003 + case["high"] * 101 + case["new_high"])
    held = [r.randint(case["low"], case["high"]) for _ in range(case["seqs"])]
    new = [r.randint(case["new_low"], case["new_high"]) for _ in range(case["seqs"])]
    new[0] = max(1, new[0])
    return held, new


# ---- inputs -------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _whole(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _frequencies(case):
    """Radians a position of every pair, in 64 bits, and the rotation's factor; with "yarn" the
    context of 32768 stretched by that factor, fast pairs left as they are."""
    n, base = case["rot"], 1e6
    i = np.arange(n // 2, dtype=np.float64)
    freq = base ** (-2.0 * i / n)
    if not case["yarn"]:
        return freq, 1.0
    at = [n * math.log(32768 / (turns * 2.0 * math.pi)) / (2.0 * math.log(base)) for turns in (32.0, 1.0)]
    low, high = max(0, math.floor(at[0])), min(n - 1, math.ceil(at[1]))
    ramp = np.clip((i - low) / max(0.001, high - low), 0.0, 1.0)
    return freq / case["yarn"] * ramp + freq * (1.0 - ramp), 0.1 * math.log(case["yarn"]) + 1.0


def _rope_inputs(case, seed):
    g = _gen(seed)
    x = _randn(g, case["rows"], case["heads"] * case["hd"])
    # a stretch of one sequence's positions, the last of them `top`
    first = max(0, case["top"] - case["rows"] - seed % 64)
    return x, torch.arange(first, first + case["rows"], dtype=torch.int32, device=DEVICE)


def _coded(x, dims):
    """Codes and scales of whole blocks, the block's values on the last two axes."""
    most = x.abs().amax(dim=dims, keepdim=True)
    e = torch.ceil(torch.log2(most.double() / MOST)).clamp(min=-100.0)
    scale = torch.exp2(e).float()
    return (x / scale).to(E4M3), scale.flatten(len(scale.shape) - len(dims))[..., 0]


def _cache_inputs(case, seed):
    """A pool of pages that other sequences have used before, its table, and the new rows."""
    g, r = _gen(seed), random.Random(seed)
    held, new = _sequences(case)
    kv, hd, page = case["kv"], case["hd"], case["page"]
    need = [-(-(a + b) // page) for a, b in zip(held, new)]
    n_pages, most = sum(need) + 3, max(need)
    names = list(range(n_pages))
    r.shuffle(names)
    table, at = np.full((case["seqs"], most), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = names[at:at + n]
        at += n
    shape = (n_pages, kv, page // BLOCK)
    k, ks = _coded(_randn(g, *shape, BLOCK, hd), (3, 4))
    v, vs = _coded(_randn(g, *shape, hd, BLOCK), (3, 4))
    rows = sum(new)
    return {"k_pages": k, "v_pages": v, "scales": torch.stack([ks, vs], -1).contiguous(),
            "table": torch.from_numpy(table).to(DEVICE), "lengths": _whole(held),
            "row_start": _whole(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)),
            "q": _randn(g, rows, case["heads"] * hd), "k": _randn(g, rows, kv * hd), "v": _randn(g, rows, kv * hd),
            "gamma": 1.0 + 0.1 * _randn(g, 2, hd), "n_pages": n_pages, "max_pages": most, "rows": rows}


def _logprob_inputs(case, seed):
    g = _gen(seed)
    x = 2.5 * _randn(g, case["rows"], case["vocab"])
    noise = torch.rand(case["rows"], case["vocab"], generator=g, device=DEVICE).clamp(min=1e-30)
    return x, (x - torch.log(-torch.log(noise) + 1e-30)).argmax(1).to(torch.int32)  # (a sampled token each)


class Rotation(ctypes.Structure):
    _fields_ = [("freqs", ctypes.c_void_p), ("n_rot", ctypes.c_int32), ("interleaved", ctypes.c_int32),
                ("magnitude", ctypes.c_float)]


class PagedCache(ctypes.Structure):
    _fields_ = [("k_pages", ctypes.c_void_p), ("v_pages", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("n_pages", ctypes.c_int32), ("page_tokens", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32)]


class PagedBatch(ctypes.Structure):
    _fields_ = [("n_seqs", ctypes.c_int32), ("n_rows", ctypes.c_int32), ("max_pages", ctypes.c_int32),
                ("row_start", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("pages", ctypes.c_void_p)]


def prepare(case, seed):
    op = case["op"]
    if op == "rope":
        x, at = _rope_inputs(case, seed)
        freq, magnitude = _frequencies(case)
        s = {"case": case, "x": x, "at": at, "out": torch.zeros_like(x), "freq": torch.from_numpy(freq).to(DEVICE),
             "magnitude": magnitude}
        s["rotation"] = Rotation(s["freq"].data_ptr(), case["rot"], case["inter"], magnitude)
        return s
    if op == "logprobs":
        x, tokens = _logprob_inputs(case, seed)
        n, top = case["rows"], case["top"]
        return {"case": case, "logits": x, "tokens": tokens, "logp": torch.zeros(n, device=DEVICE),
                "entropy": torch.zeros(n, device=DEVICE),
                "top": torch.zeros(n, top, dtype=torch.int32, device=DEVICE),
                "top_logp": torch.zeros(n, top, device=DEVICE)}
    s = _cache_inputs(case, seed) | {"case": case}
    s["out"] = torch.zeros_like(s["q"])
    s["cache"] = PagedCache(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["scales"].data_ptr(), s["n_pages"],
                            case["page"], case["kv"], case["hd"])
    s["batch"] = PagedBatch(case["seqs"], s["rows"], s["max_pages"], s["row_start"].data_ptr(),
                            s["lengths"].data_ptr(), s["table"].data_ptr())
    if op == "append":
        freq, magnitude = _frequencies(case)
        s |= {"freq": torch.from_numpy(freq).to(DEVICE), "magnitude": magnitude}
        s["rotation"] = Rotation(s["freq"].data_ptr(), case["rot"], case["inter"], magnitude)
    return s


# ---- one pass -------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


def _run_own(case, s):
    lib = importlib.import_module("gnc-x_amd").load()
    op, ref = case["op"], ctypes.byref
    if op == "rope":
        width = case["heads"] * case["hd"]
        lib.gncx_hip_rope_rows(s["x"].data_ptr(), case["rows"], width, case["heads"], case["hd"], s["at"].data_ptr(),
                               ref(s["rotation"]), width, s["out"].data_ptr())
        return s["out"]
    if op == "logprobs":
        lib.gncx_hip_token_logprobs(s["logits"].data_ptr(), case["rows"], case["vocab"], s["tokens"].data_ptr(),
                                    case["top"], s["logp"].data_ptr(), s["entropy"].data_ptr(),
                                    s["top"].data_ptr() if case["top"] else None,
                                    s["top_logp"].data_ptr() if case["top"] else None)
        return {"logp": s["logp"], "entropy": s["entropy"], "top": s["top"], "top_logp": s["top_logp"]}
    if op == "append":
        lib.gncx_hip_kv_append_paged(ref(s["cache"]), ref(s["batch"]), s["q"].data_ptr(), s["k"].data_ptr(),
                                     s["v"].data_ptr(), case["heads"], s["gamma"].data_ptr(), 0, 4 * case["hd"],
                                     case["norm"], EPS, ref(s["rotation"]), s["out"].data_ptr())
        return {"q": s["out"], "k": s["k_pages"], "v": s["v_pages"], "scales": s["scales"]}
    lib.gncx_hip_attention_paged(ref(s["cache"]), ref(s["batch"]), s["q"].data_ptr(), case["heads"],
                                 1.0 / math.sqrt(case["hd"]), case["sw"], s["out"].data_ptr())
    return s["out"]


def _run_plain(case, s):
    op = case["op"]
    if op == "rope":
        x = s["x"].view(case["rows"], case["heads"], case["hd"])
        s["out"].copy_(_plain_rotated(x, s["at"], s).view(case["rows"], -1))
        return s["out"]
    if op == "append":
        return _plain_append(case, s)
    if op == "attend":
        return _plain_attend(case, s)
    return _plain_logprobs(case, s)


def _plain_rotated(x, at, s):
    """x [rows][heads][head_dim], angles in 64 bits."""
    n, inter = s["case"]["rot"], s["case"]["inter"]
    angle = at.double().unsqueeze(1) * s["freq"]
    c, d = ((f(angle) * s["magnitude"]).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if inter else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a * c - b * d, b * c + a * d
    turned = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., n:]], -1)


def _plain_head(x, gamma, at, s):
    norm = s["case"]["norm"]
    if norm >= 0:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    if norm > 0:
        x = x * gamma
    return _plain_rotated(x, at, s)


def _plain_places(s):
    """Of every row: its sequence and its position."""
    row = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["row_start"].long(), row, right=True) - 1
    return seq, s["lengths"].long()[seq] + row - s["row_start"].long()[seq]


def _plain_append(case, s):
    kv, hd, page, h = case["kv"], case["hd"], case["page"], case["heads"]
    seq, at = _plain_places(s)
    s["out"].copy_(_plain_head(s["q"].view(-1, h, hd), s["gamma"][0], at, s).view(-1, h * hd))
    k = _plain_head(s["k"].view(-1, kv, hd), s["gamma"][1], at, s)
    v = s["v"].view(-1, kv, hd)
    name, block, place = s["table"][seq, at // page].long(), at % page // BLOCK, at % BLOCK
    # which tokens a block held before, and whose codes move to a larger scale
    before = torch.minimum(s["lengths"].long()[seq] - (at - place), place)
    where = name * (page // BLOCK) + block
    for x, codes, i, flat in ((k, s["k_pages"], 0, (-2, -1)), (v, s["v_pages"], 1, (-1, -2))):
        n_blocks = codes.shape[0] * codes.shape[2]
        most = torch.zeros(n_blocks, kv, device=DEVICE).scatter_reduce_(0, where.unsqueeze(1).expand(-1, kv),
                                                                        x.abs().amax(-1), "amax")[where]
        # the least power of two that 448 times reaches it
        m, e = torch.frexp(most / MOST)
        e = torch.where(most == 0, -100, torch.where(m == 0.5, e - 1, e)).clamp(min=-100)
        scale = torch.ldexp(torch.ones_like(most), e)
        old = s["scales"][name, :, block, i]
        held = (before > 0).unsqueeze(1)
        scale = torch.where(held, torch.maximum(old, scale), scale)
        all_codes = codes[name, :, block].float()  # [rows][kv] blocks
        if i:
            all_codes = all_codes.transpose(-2, -1)
        token = torch.arange(BLOCK, device=DEVICE).view(1, 1, BLOCK, 1)
        moved = (all_codes * (old / scale).view(-1, kv, 1, 1)).to(E4M3).float()
        all_codes = torch.where((token < before.view(-1, 1, 1, 1)) & held.view(-1, 1, 1, 1), moved, all_codes)
        if i:
            all_codes = all_codes.transpose(-2, -1)
        codes[name, :, block] = all_codes.to(E4M3)
        s["scales"][name, :, block, i] = scale
        new = (x / scale.unsqueeze(-1)).to(E4M3)
        if i:
            codes[name, :, block, :, place] = new
        else:
            codes[name, :, block, place] = new
    return {"q": s["out"], "k": s["k_pages"], "v": s["v_pages"], "scales": s["scales"]}


def _plain_attend(case, s):
    kv, hd, page, h, sw = case["kv"], case["hd"], case["page"], case["heads"], case["sw"]
    g, seqs = h // kv, case["seqs"]
    names = s["table"].clamp(min=0).long()  # [seqs][max_pages]
    keys = s["k_pages"][names].float() * s["scales"][names][..., 0, None, None]
    vals = s["v_pages"][names].float() * s["scales"][names][..., 1, None, None]
    keys = keys.permute(0, 2, 5, 1, 3, 4).reshape(seqs, kv, hd, -1)
    vals = vals.permute(0, 2, 1, 3, 5, 4).reshape(seqs, kv, -1, hd)
    seq, at = _plain_places(s)
    inside = torch.arange(s["rows"], device=DEVICE) - s["row_start"].long()[seq]
    t, most = case["new_high"], keys.shape[-1]
    q = torch.zeros(seqs, t, h * hd, device=DEVICE)
    q[seq, inside] = s["q"]
    place = torch.full((seqs, t), -1, device=DEVICE)
    place[seq, inside] = at
    q = q.view(seqs, t, kv, g, hd).transpose(1, 2).reshape(seqs, kv, t * g, hd)
    key = torch.arange(most, device=DEVICE)
    seen = key <= place.unsqueeze(-1)
    if sw:
        seen = seen & (key > place.unsqueeze(-1) - sw)
    score = (torch.matmul(q, keys) / math.sqrt(hd)).view(seqs, kv, t, g, most)
    score = torch.where(seen.view(seqs, 1, t, 1, most), score, -INF)
    w = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(seqs, kv, t * g, most), vals).view(seqs, kv, t, g, hd) / total
    s["out"].copy_(out.permute(0, 2, 1, 3, 4).reshape(seqs, t, h * hd)[seq, inside])
    return s["out"]


def _plain_logprobs(case, s):
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    norm = torch.log(total)
    s["logp"].copy_((x.gather(1, s["tokens"].long().unsqueeze(1)) - top - norm)[:, 0])
    s["entropy"].copy_((norm - (e * (x - top)).sum(1, keepdim=True) / total)[:, 0])
    if case["top"]:
        # equal logits by the lowest word: the float's bits in the floats' order, then the word
        bits = s["logits"].view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * 2 ** 32 - torch.arange(case["vocab"], device=DEVICE)
        best = torch.topk(order, case["top"], dim=1).indices
        s["top"].copy_(best)
        s["top_logp"].copy_(x.gather(1, best) - top - norm)
    return {"logp": s["logp"], "entropy": s["entropy"], "top": s["top"], "top_logp": s["top_logp"]}


# ---- what a pass cannot do without ---------------------------------------------
def work(case):
    op = case["op"]
    if op == "rope":
        floats = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 8 * floats + 4 * case["rows"] + 4 * case["rot"],
                "flops": 3 * case["rows"] * case["heads"] * case["rot"]}
    if op == "logprobs":
        cells = case["rows"] * case["vocab"]
        return {"bytes": 4 * cells + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * cells}
    held, new = _sequences(case)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    if op == "append":
        rows, blocks, before = sum(new), 0, 0
        for a, n in zip(held, new):
            if n:
                blocks += (a + n - 1) // BLOCK - a // BLOCK + 1
                before += a % BLOCK
        # q read and written, k and v read, a byte written for each, scales
        return {"bytes": 8 * rows * h * hd + 10 * rows * kv * hd + 8 * kv * blocks, "flops": 10 * rows * (h + kv) * hd}
    sw, tokens, pairs = case["sw"], 0, 0
    for a, n in zip(held, new):
        if not n:
            continue
        low = max(0, a - sw + 1) if sw else 0
        tokens += a + n - low
        at = np.arange(a, a + n, dtype=np.int64)
        pairs += int((np.minimum(at + 1, sw) if sw else at + 1).sum())
    return {"bytes": kv * tokens * 2 * hd + kv * tokens * 8 // BLOCK + 8 * sum(new) * h * hd, "flops": 4 * h * hd * pairs}


# ---- 64-bit references -----------------------------------------------------------
def _exact_turned(case, x, at):
    """x [rows][heads][head_dim] in 64 bits, as complex numbers turned."""
    freq, magnitude = _frequencies(case)
    n = case["rot"]
    turn = torch.from_numpy(np.exp(1j * (at.cpu().numpy().astype(np.float64)[:, None] * freq)) * magnitude).to(DEVICE)
    y = x.clone()
    if case["inter"]:
        z = torch.view_as_complex(x[..., :n].reshape(*x.shape[:-1], n // 2, 2).contiguous()) * turn[:, None, :]
        y[..., :n] = torch.view_as_real(z).reshape(*x.shape[:-1], n)
    else:
        z = torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous()) * turn[:, None, :]
        y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
    return y


def _exact_e4m3(x):
    """The nearest e4m3 values, ties to even: steps of 2^(e - 3), e at least -6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(x / step) * step


def _exact_append(case, seed):
    s = _cache_inputs(case, seed)
    held, new = _sequences(case)
    kv, hd, page, h = case["kv"], case["hd"], case["page"], case["heads"]
    at = torch.cat([torch.arange(a, a + n) for a, n in zip(held, new)]).to(DEVICE)

    def head(x, n, gamma):
        x = x.double().view(-1, n, hd)
        if case["norm"] >= 0:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPS)
        return _exact_turned(case, x * gamma.double() if case["norm"] > 0 else x, at)

    q, rows = head(s["q"], h, s["gamma"][0]), {"k": head(s["k"], kv, s["gamma"][1]), "v": s["v"].double().view(-1, kv, hd)}
    codes = {"k": s["k_pages"].double(), "v": s["v_pages"].double().transpose(-2, -1).contiguous()}
    scales, table, first = s["scales"].double(), s["table"].cpu().numpy(), 0
    for i, (a, n) in enumerate(zip(held, new)):
        p = a
        while p < a + n:
            end = min(a + n, (p // BLOCK + 1) * BLOCK)
            name, block, lo, hi = int(table[i, p // page]), p % page // BLOCK, p % BLOCK, p % BLOCK + end - p
            for j, which in enumerate("kv"):
                x = rows[which][first + p - a:first + end - a].transpose(0, 1)  # [kv][tokens][hd]
                most = x.abs().amax((1, 2))
                scale = torch.exp2(torch.ceil(torch.log2(most / MOST))).clamp(min=LEAST_SCALE)
                if lo:
                    was = scales[name, :, block, j]
                    scale = torch.maximum(was, scale)
                    codes[which][name, :, block, :lo] = _exact_e4m3(codes[which][name, :, block, :lo] * (was / scale)[:, None, None])
                codes[which][name, :, block, lo:hi] = _exact_e4m3(x / scale[:, None, None])
                scales[name, :, block, j] = scale
            p = end
        first += n
    return {"q": q.reshape(-1, h * hd), "k": codes["k"], "v": codes["v"].transpose(-2, -1).contiguous(), "scales": scales}


def _exact_attend(case, seed):
    s = _cache_inputs(case, seed)
    held, new = _sequences(case)
    kv, hd, h, sw = case["kv"], case["hd"], case["heads"], case["sw"]
    out, first, g = torch.empty(s["rows"], h, hd, dtype=torch.float64, device=DEVICE), 0, h // kv
    for i, (a, n) in enumerate(zip(held, new)):
        if not n:
            continue
        names = s["table"][i, :-(-(a + n) // case["page"])].long()
        at = torch.arange(a, a + n, device=DEVICE)
        key = torch.arange(a + n, device=DEVICE)
        hidden = key[None, :] > at[:, None]
        if sw:
            hidden |= key[None, :] <= at[:, None] - sw
        for b in range(kv):
            scale = s["scales"][names, b].double()
            k = (s["k_pages"][names, b].double() * scale[..., 0, None, None]).reshape(-1, hd)[:a + n]
            v = (s["v_pages"][names, b].double() * scale[..., 1, None, None]).transpose(-2, -1).reshape(-1, hd)[:a + n]
            for j in range(b * g, b * g + g):
                q = s["q"][first:first + n, j * hd:(j + 1) * hd].double()
                score = (q @ k.t().contiguous() / math.sqrt(hd)).masked_fill(hidden, -INF)
                out[first:first + n, j] = torch.softmax(score, 1) @ v
        first += n
    return out.view(s["rows"], h * hd)


def exact(case, seed):
    op = case["op"]
    if op == "rope":
        x, at = _rope_inputs(case, seed)
        return _exact_turned(case, x.double().view(case["rows"], case["heads"], case["hd"]), at).view(case["rows"], -1)
    if op == "append":
        return _exact_append(case, seed)
    if op == "attend":
        return _exact_attend(case, seed)
    x, tokens = _logprob_inputs(case, seed)
    logp = torch.log_softmax(x.double(), 1)
    best = torch.sort(x, dim=1, descending=True).values[:, :case["top"]]
    return {"logp": logp.gather(1, tokens.long()[:, None])[:, 0], "entropy": -(logp.exp() * logp).sum(1), "top": None,
            "top_logp": best.double() - torch.logsumexp(x.double(), 1, keepdim=True)}
