"""The operators for several candidate continuations of one sequence, over the
cases a user of them meets: attention for a tree of drafted tokens, keeping the
accepted rows of the caches, beam search's selection, and the reordering of the
beams' caches.

  listed()              the named cases
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   inputs and buffers on the GPU
  run(state)            one pass, its outputs: the library's entry points where
                        own is true, elementary torch operations otherwise
  work(case)            bytes and operations a pass cannot do without
  exact(case, seed)     the outputs in 64 bits, written apart from run()

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

EPS = 1e-6
ROPE_BASE = 1e6
INF = math.inf


# ---- the cases ----------------------------------------------------------------
def listed():
    return [
        # a linear draft of four tokens after a short prompt: the smallest verification, all latency
        {"name": "tree_chain_4_at_300", "op": "tree", "shape": "chain", "nodes": 4, "heads": 32, "kv": 8, "hd": 128,
         "pos": 300, "sw": 0, "norm": 1},
        # an ordinary draft tree in a medium conversation
        {"name": "tree_16_at_2048", "op": "tree", "shape": "binary", "nodes": 16, "heads": 32, "kv": 8, "hd": 128,
         "pos": 2048, "sw": 0, "norm": 1},
        # a wide draft tree over a longer one, a model with four KV heads
        {"name": "tree_128_at_8192", "op": "tree", "shape": "wide", "nodes": 128, "heads": 32, "kv": 4, "hd": 128,
         "pos": 8192, "sw": 0, "norm": 1},
        # an odd tree over a long document, a model without the per-head norms
        {"name": "tree_25_at_32749", "op": "tree", "shape": "random", "nodes": 25, "heads": 32, "kv": 8, "hd": 128,
         "pos": 32749, "sw": 0, "norm": -1},
        # many candidates at once, 64-wide heads without groups, a sliding window
        {"name": "tree_400_at_4001", "op": "tree", "shape": "random", "nodes": 400, "heads": 16, "kv": 16, "hd": 64,
         "pos": 4001, "sw": 2048, "norm": 1},
        # the accepted path of a 16-node draft in the caches of a 36-layer model
        {"name": "keep_4_of_16", "op": "keep", "layers": 36, "kv_dim": 1024, "pos": 2048, "nodes": 16, "rows": 4},
        # a long linear draft, mostly accepted, four KV heads
        {"name": "keep_101_of_256", "op": "keep", "layers": 36, "kv_dim": 512, "pos": 1000, "nodes": 256,
         "rows": 101},
        # a small beam over a 32000-word vocabulary
        {"name": "beam_4_x_32000", "op": "beam", "beams": 4, "vocab": 32000, "out": 8, "finished": 0, "masked": 0},
        # a wide beam over a large vocabulary
        {"name": "beam_16_x_151936", "op": "beam", "beams": 16, "vocab": 151936, "out": 32, "finished": 0,
         "masked": 0},
        # constrained decoding (most words masked), an odd vocabulary, two beams already finished
        {"name": "beam_5_x_50257_masked", "op": "beam", "beams": 5, "vocab": 50257, "out": 5, "finished": 2,
         "masked": 1},
        # the generated rows of four beams, 36 layers
        {"name": "reorder_4_x_100", "op": "reorder", "layers": 36, "beams": 4, "kv_dim": 1024, "row0": 500,
         "rows": 100},
        # eight beams with long continuations
        {"name": "reorder_8_x_1000", "op": "reorder", "layers": 12, "beams": 8, "kv_dim": 1024, "row0": 33,
         "rows": 1000},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_PAIRS = 128 * 32 * 8320 * 128  # of a drawn tree: nodes x heads x keys x head_dim


def draw(rng):
    op = rng.choice(["tree"] * 5 + ["keep"] * 2 + ["beam"] * 3 + ["reorder"] * 2)
    if op == "tree":
        h, kv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (32, 4, 128), (64, 8, 128), (32, 1, 128), (16, 16, 64),
                                (32, 8, 64), (8, 2, 256), (12, 4, 128)])
        n, pos = _log(rng, 1, 512), _log(rng, 1, 32768)
        pos = max(1, min(pos, MOST_PAIRS // (n * h * hd) - n))
        return {"op": op, "shape": rng.choice(["chain", "binary", "wide", "random"]), "nodes": n, "heads": h,
                "kv": kv, "hd": hd, "pos": pos, "sw": rng.choice([0, 0, 0, 512, 1024]), "norm": rng.choice([1, 1, -1])}
    if op == "keep":
        n = _log(rng, 1, 512)
        return {"op": op, "layers": _log(rng, 1, 48), "kv_dim": rng.choice([128, 256, 512, 1024, 2048]),
                "pos": _log(rng, 1, 4096), "nodes": n, "rows": rng.randint(1, n)}
    if op == "beam":
        b = _log(rng, 1, 32)
        return {"op": op, "beams": b, "vocab": _log(rng, 300, 256000), "out": rng.choice([b, 2 * b]),
                "finished": rng.choice([0, 0, b // 3]), "masked": rng.choice([0, 0, 1])}
    b, layers, d = _log(rng, 2, 32), _log(rng, 1, 48), rng.choice([128, 512, 1024, 2048])
    most = 12 * 8 * 1000 * 1024 // (b * layers * d)
    return {"op": op, "layers": layers, "beams": b, "kv_dim": d, "row0": _log(rng, 1, 600),
            "rows": _log(rng, 1, max(1, most))}


# ---- inputs -------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _parents(case):
    """The draft tree of a case (a drafting program keeps its shape)."""
    n, shape = case["nodes"], case["shape"]
    if shape != "random":
        arity = {"chain": 1, "binary": 2, "wide": 4}[shape]
        return [(i - 1) // arity if i else -1 for i in range(n)]
    r = random.Random(n)
    return [-1 if i == 0 or r.random() < 0.05 else r.randrange(max(0, i - 12), i) for i in range(n)]


def _tree(case):
    """Each node's depth, and which nodes it sees: its ancestors and itself."""
    depth, sees = [], np.eye(case["nodes"], dtype=bool)
    for i, p in enumerate(_parents(case)):
        depth.append(depth[p] + 1 if p >= 0 else 0)
        if p >= 0:
            sees[i] |= sees[p]
    return depth, sees


def _tree_inputs(case, seed):
    g = _gen(seed)
    n, h, kv, hd = case["nodes"], case["heads"], case["kv"], case["hd"]
    rows = case["pos"] + n
    gamma = 1.0 + 0.1 * _randn(g, 2, hd)
    return (_randn(g, n, h * hd), _randn(g, n, kv * hd), _randn(g, n, kv * hd), _randn(g, rows, kv * hd),
            _randn(g, rows, kv * hd), gamma)


def _keep_inputs(case, seed):
    g = _gen(seed)
    shape = (case["layers"], case["pos"] + case["nodes"], case["kv_dim"])
    rows = sorted(random.Random(seed).sample(range(case["nodes"]), case["rows"]))
    return _randn(g, *shape), _randn(g, *shape), rows


def _beam_inputs(case, seed):
    g = _gen(seed)
    b, v = case["beams"], case["vocab"]
    logits = 2.5 * _randn(g, b, v)
    if case["masked"]:  # a grammar that leaves one word in fifty
        logits.masked_fill_(torch.rand(b, v, generator=g, device="cuda") > 0.02, -INF)
    scores = -20.0 + _randn(g, b)
    finished = (torch.randperm(b, generator=g, device="cuda") < case["finished"]).to(torch.int32)
    return logits, scores, finished


def _reorder_inputs(case, seed):
    g = _gen(seed)
    shape = (case["layers"], case["beams"], case["row0"] + case["rows"], case["kv_dim"])
    # the parents of a step: a few good beams continue several times
    pick = torch.rand(case["beams"], generator=g, device="cuda").square() * case["beams"]
    return _randn(g, *shape), _randn(g, *shape), pick.to(torch.int32)


def _layers(cache):
    """The address of every layer's cache, as the entry points take them."""
    step, base = cache.stride(0) * cache.element_size(), cache.data_ptr()
    return (ctypes.c_void_p * cache.shape[0])(*range(base, base + cache.shape[0] * step, step))


def prepare(case, seed):
    op = case["op"]
    if op == "tree":
        q, k, v, kc, vc, gamma = _tree_inputs(case, seed)
        depth, sees = _tree(case)
        half = case["hd"] // 2
        # the rotation's frequencies in float32, as the other entry points have them
        freq = np.float32(1) / np.power(ROPE_BASE, (np.arange(half, dtype=np.float32) * 2 / np.float32(2 * half))
                                        .astype(np.float64)).astype(np.float32)
        return {"case": case, "q": q, "k": k, "v": v, "kc": kc, "vc": vc, "gamma": gamma, "out": torch.zeros_like(q),
                "parents": np.array(_parents(case), np.int32), "depth": torch.tensor(depth, device="cuda"),
                "sees": torch.from_numpy(sees).cuda(), "freq": torch.from_numpy(freq).cuda()}
    if op == "keep":
        kc, vc, rows = _keep_inputs(case, seed)
        return {"case": case, "kc": kc, "vc": vc, "layers": (_layers(kc), _layers(vc)),
                "rows": np.array(rows, np.int32), "index": torch.tensor(rows, device="cuda")}
    if op == "beam":
        logits, scores, finished = _beam_inputs(case, seed)
        whole = dict(dtype=torch.int32, device="cuda")
        return {"case": case, "logits": logits, "scores": scores, "finished": finished,
                "parents": torch.zeros(case["out"], **whole), "tokens": torch.zeros(case["out"], **whole),
                "best": torch.zeros(case["out"], device="cuda")}
    kc, vc, parents = _reorder_inputs(case, seed)
    return {"case": case, "kc": kc, "vc": vc, "layers": (_layers(kc), _layers(vc)), "parents": parents}


# ---- one pass -------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


def _run_own(case, s):
    lib = importlib.import_module("gnc-x_amd").load()
    op = case["op"]
    if op == "tree":
        hd, norm = case["hd"], case["norm"]
        lib.gncx_hip_attention_tree(
            s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["kc"].data_ptr(), s["vc"].data_ptr(),
            case["pos"], case["nodes"], s["parents"].ctypes.data, case["heads"], case["kv"], hd, 1.0 / math.sqrt(hd),
            case["sw"], s["gamma"].data_ptr(), 0, 4 * hd, norm, EPS, 0, 0, ROPE_BASE, s["out"].data_ptr())
        return {"out": s["out"], "q": s["q"], "k": s["k"], "k_rows": s["kc"][case["pos"]:],
                "v_rows": s["vc"][case["pos"]:]}
    if op == "keep":
        lib.gncx_hip_kv_keep_rows(*s["layers"], case["layers"], case["kv_dim"], case["pos"],
                                  s["rows"].ctypes.data, case["rows"])
        return {"kc": s["kc"], "vc": s["vc"]}
    if op == "beam":
        lib.gncx_hip_beam_select(s["logits"].data_ptr(), case["beams"], case["vocab"], s["scores"].data_ptr(),
                                 s["finished"].data_ptr(), 2, case["out"], s["parents"].data_ptr(),
                                 s["tokens"].data_ptr(), s["best"].data_ptr())
        return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["best"]}
    lib.gncx_hip_kv_reorder(*s["layers"], case["layers"], case["beams"], s["kc"].stride(1), case["kv_dim"],
                            case["row0"], case["rows"], s["parents"].data_ptr())
    return {"kc": s["kc"], "vc": s["vc"]}


def _run_plain(case, s):
    op = case["op"]
    if op == "tree":
        return _plain_tree(case, s)
    if op == "keep":
        at = case["pos"] + s["index"]
        s["kc"][:, case["pos"]:case["pos"] + case["rows"]] = s["kc"][:, at]
        s["vc"][:, case["pos"]:case["pos"] + case["rows"]] = s["vc"][:, at]
        return {"kc": s["kc"], "vc": s["vc"]}
    if op == "beam":
        return _plain_beam(case, s)
    parents, end = s["parents"].long(), case["row0"] + case["rows"]
    s["kc"][:, :, case["row0"]:end] = s["kc"][:, parents, case["row0"]:end]
    s["vc"][:, :, case["row0"]:end] = s["vc"][:, parents, case["row0"]:end]
    return {"kc": s["kc"], "vc": s["vc"]}


def _plain_prologue(x, gamma, angle, norm):
    if norm > 0:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma
    half = x.shape[-1] // 2
    c, s = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_tree(case, s):
    n, h, kv, hd, pos, sw = (case[x] for x in ("nodes", "heads", "kv", "hd", "pos", "sw"))
    g, at = h // kv, pos + s["depth"]
    # float32 angles, as the decode step has them; their cosines in 64 bits
    angle = (at.float().unsqueeze(1) * s["freq"]).double()
    s["q"].copy_(_plain_prologue(s["q"].view(n, h, hd), s["gamma"][0], angle, case["norm"]).view(n, h * hd))
    s["k"].copy_(_plain_prologue(s["k"].view(n, kv, hd), s["gamma"][1], angle, case["norm"]).view(n, kv * hd))
    s["kc"][pos:pos + n] = s["k"]
    s["vc"][pos:pos + n] = s["v"]
    first = max(0, pos - sw + 1) if sw else 0
    q = s["q"].view(n, kv, g, hd).transpose(0, 1).reshape(kv, n * g, hd)
    keys = s["kc"][first:].view(-1, kv, hd).permute(1, 2, 0).contiguous()
    vals = s["vc"][first:].view(-1, kv, hd).transpose(0, 1).contiguous()
    cached = torch.arange(first, pos, device="cuda")
    visible = torch.cat([torch.ones(n, pos - first, dtype=torch.bool, device="cuda"), s["sees"]], 1)
    if sw:
        visible = visible & (torch.cat([cached, at]).unsqueeze(0) > (at - sw).unsqueeze(1))
    score = torch.matmul(q, keys).view(kv, n, g, -1) / math.sqrt(hd)
    score = torch.where(visible.unsqueeze(1).unsqueeze(0), score, -INF)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True) + 1e-12
    out = torch.matmul(w.view(kv, n * g, -1), vals).view(kv, n, g, hd) / total
    s["out"].copy_(out.transpose(0, 1).reshape(n, h * hd))
    return {"out": s["out"], "q": s["q"], "k": s["k"], "k_rows": s["kc"][pos:], "v_rows": s["vc"][pos:]}


def _plain_beam(case, s):
    b, v, n = case["beams"], case["vocab"], case["out"]
    x = s["logits"].double()  # 64 bits: the order of near candidates of different beams
    top = x.amax(1, keepdim=True).clamp(min=-1e300)  # (a beam with every word masked)
    logp = x - (top + torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    logp = torch.where(x == -INF, -INF, logp)
    score = s["scores"].double().unsqueeze(1) + logp
    done = torch.full_like(score, -INF)
    done[:, 2] = s["scores"].double()
    score = torch.where(s["finished"].bool().unsqueeze(1), done, score).view(-1)
    # the n best, equal ones by the lowest index
    least = torch.topk(score, n).values[n - 1]
    among = torch.nonzero(score >= least).view(-1)
    best, order = torch.sort(score[among], descending=True, stable=True)
    index, best = among[order[:n]], best[:n]
    none = best == -INF
    s["parents"].copy_(torch.where(none, -1, index // v))
    s["tokens"].copy_(torch.where(none, -1, index % v))
    s["best"].copy_(best)
    return {"parents": s["parents"], "tokens": s["tokens"], "scores": s["best"]}


# ---- what a pass cannot do without ---------------------------------------------
def work(case):
    op = case["op"]
    if op == "tree":
        n, h, kv, hd, pos, sw = (case[x] for x in ("nodes", "heads", "kv", "hd", "pos", "sw"))
        depth, sees = _tree(case)
        at = pos + np.array(depth)
        low = np.maximum(0, at - sw + 1) if sw else np.zeros(n, np.int64)
        pairs = int(np.maximum(0, pos - low).sum() + (sees & (at[None, :] >= low[:, None])).sum())
        rows = pos - int(low.min()) if int(low.min()) < pos else 0
        return {"bytes": 8 * kv * hd * rows + 12 * n * h * hd + 20 * n * kv * hd, "flops": 4 * h * hd * pairs}
    if op == "keep":
        return {"bytes": 16 * case["layers"] * case["rows"] * case["kv_dim"], "flops": 0}
    if op == "beam":
        cells = (case["beams"] - case["finished"]) * case["vocab"]
        return {"bytes": 4 * cells + 12 * (case["beams"] + case["out"]), "flops": 4 * cells}
    # expected: each beam that moves is written, each that another continues from is read
    b = case["beams"]
    chosen = np.diff(np.sqrt(np.arange(b + 1) / b))
    moved = b - 1 + float((1 - (1 - chosen) ** (b - 1)).sum())
    return {"bytes": 8 * case["layers"] * moved * case["rows"] * case["kv_dim"], "flops": 0}


# ---- 64-bit references -----------------------------------------------------------
def _exact_tree(case, seed):
    q, k, v, kc, vc, gamma = (a.double() for a in _tree_inputs(case, seed))
    n, h, kv, hd, pos, sw = (case[x] for x in ("nodes", "heads", "kv", "hd", "pos", "sw"))
    parents, g = _parents(case), h // kv
    path = []  # of every node: its ancestors from the root on, and itself
    for i, p in enumerate(parents):
        path.append((path[p] if p >= 0 else []) + [i])
    at = np.array([pos + len(p) - 1 for p in path])
    exponent = (np.float32(2) * np.arange(hd // 2, dtype=np.float32) / np.float32(hd)).astype(np.float64)
    freq = np.float32(1) / (ROPE_BASE ** exponent).astype(np.float32)
    turn = torch.from_numpy((at.astype(np.float32)[:, None] * freq[None, :]).astype(np.float64)).cuda()
    turn = torch.polar(torch.ones_like(turn), turn)[:, None, :]

    def rotated(x, heads, weight):
        x = x.view(n, heads, hd)
        if case["norm"] > 0:
            x = x / torch.sqrt((x * x).sum(2, keepdim=True) / hd + EPS) * weight
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], 2).reshape(n, heads * hd)

    q, k = rotated(q, h, gamma[0]), rotated(k, kv, gamma[1])
    kc[pos:], vc[pos:] = k, v
    hidden = torch.ones(n, pos + n, dtype=torch.bool)
    for i, p in enumerate(path):
        low = max(0, at[i] - sw + 1) if sw else 0
        hidden[i, low:pos] = False
        hidden[i, [pos + a for a in p if at[a] >= low]] = False
    hidden, out = hidden.cuda(), torch.empty_like(q)
    for i in range(h):
        mine, theirs = slice(i * hd, (i + 1) * hd), slice(i // g * hd, (i // g + 1) * hd)
        score = q[:, mine].contiguous() @ kc[:, theirs].t().contiguous() / math.sqrt(hd)
        out[:, mine] = torch.softmax(score.masked_fill(hidden, -INF), 1) @ vc[:, theirs].contiguous()
    return {"out": out, "q": q, "k": k, "k_rows": k, "v_rows": v}


def exact(case, seed):
    op = case["op"]
    if op == "tree":
        return _exact_tree(case, seed)
    if op == "beam":
        logits, scores, finished = _beam_inputs(case, seed)
        b, v, n = case["beams"], case["vocab"], case["out"]
        logp = torch.log_softmax(logits.double(), 1).nan_to_num(nan=-INF).cpu().numpy()
        total = scores.double().cpu().numpy()[:, None] + logp
        for i in np.flatnonzero(finished.cpu().numpy()):
            total[i] = -INF
            total[i, 2] = float(scores[i])
        flat = total.reshape(-1)
        best = flat[np.argsort(-flat, kind="stable")[:n]]
        return {"parents": None, "tokens": None, "scores": torch.from_numpy(best)}
    if op == "keep":
        kc, vc, rows = _keep_inputs(case, seed)
    else:
        kc, vc, parents = _reorder_inputs(case, seed)
    both = []
    for c in (kc, vc):
        c = c.double()
        if op == "keep":
            old = c.clone()
            for i, r in enumerate(rows):
                c[:, case["pos"] + i] = old[:, case["pos"] + r]
        else:
            rows, old = slice(case["row0"], case["row0"] + case["rows"]), c.clone()
            for i, p in enumerate(parents.tolist()):
                c[:, i, rows] = old[:, p, rows]
        both.append(c)
    return {"kc": both[0], "vc": both[1]}
