"""Cases and plain forms of the operators of a drafted-token decoding step over a K/V cache.

Four operators, one pass of each:
  cache      new K/V rows are quantised into the cache (one fp32 scale per row) and read back
  attention  the queries of a tree of drafted tokens over the cached positions and their own branch
  verify     the walk down the tree: which drafted tokens the target model keeps, and the token after them
  keep       the kept branch's cache rows move up behind the context

With `own` false, run() computes in elementary torch operations; with `own` true it calls the
library's entry points on the same state.
"""
import importlib.util
import math
import os

import numpy as np
import torch

own = False

VOCAB = 151936       # the model's vocabulary
CAPACITY = 8192      # positions of a cache slot
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "int8": 1}
TOP = {"e4m3": 448.0, "int8": 127.0}

_qb = None


def _library():
    global _qb
    if _qb is None:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location("qwen_b200", os.path.join(here, "qwen600-rocm-inference_b200", "qwen_b200.py"))
        _qb = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_qb)
    return _qb


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a full batch: a token's K and V rows per sequence into an e4m3 cache
        {"name": "cache step 128", "op": "cache", "b": 128, "t": 1, "kv": 8, "dim": 128, "store": "e4m3", "src": "bf16", "dst": "bf16", "cap": 1024},
        # prompts of 16 sequences entering an int8 cache
        {"name": "cache prompts 16x2048", "op": "cache", "b": 16, "t": 2048, "kv": 8, "dim": 128, "store": "int8", "src": "bf16", "dst": "bf16", "cap": 4096},
        # odd sizes, fp32 projections, heads of 64
        {"name": "cache odd fp32", "op": "cache", "b": 3, "t": 517, "kv": 5, "dim": 64, "store": "e4m3", "src": "fp32", "dst": "fp32", "cap": 1031},
        # one token of one sequence: the latency of plain decoding
        {"name": "attention 1x1 at 1024", "op": "attention", "b": 1, "t": 1, "kv": 8, "group": 2, "dim": 128, "q": "bf16", "store": "bf16", "len": 1024, "ragged": False, "shape": "chain"},
        # one sequence, a full tree of 64 nodes at the end of a slot
        {"name": "attention 1x64 at 8128", "op": "attention", "b": 1, "t": 64, "kv": 8, "group": 2, "dim": 128, "q": "bf16", "store": "bf16", "len": 8128, "ragged": False, "shape": "tree"},
        # a batch of short chains over ragged int8 caches, heads of 64
        {"name": "attention 32x7 int8", "op": "attention", "b": 32, "t": 7, "kv": 4, "group": 4, "dim": 64, "q": "fp16", "store": "int8", "len": 4099, "ragged": True, "shape": "chain"},
        # serving: 128 sequences, small trees over ragged e4m3 caches
        {"name": "attention 128x8 e4m3", "op": "attention", "b": 128, "t": 8, "kv": 8, "group": 2, "dim": 128, "q": "bf16", "store": "e4m3", "len": 8184, "ragged": True, "shape": "tree"},
        # many query heads on each K/V head and full trees: bound by arithmetic
        {"name": "attention 8x64 group 8", "op": "attention", "b": 8, "t": 64, "kv": 8, "group": 8, "dim": 128, "q": "bf16", "store": "bf16", "len": 8128, "ragged": True, "shape": "tree"},
        # one sequence, a chain of seven drafted tokens (their drafter gives no probabilities)
        {"name": "verify 1x8", "op": "verify", "b": 1, "t": 8, "vocab": VOCAB, "type": "fp32", "draft": False, "shape": "chain", "temp": 0.6},
        # 32 sequences, chains drafted from a small model's distribution
        {"name": "verify 32x8 drafted", "op": "verify", "b": 32, "t": 8, "vocab": VOCAB, "type": "fp32", "draft": True, "shape": "chain", "temp": 1.0},
        # the accepted rows of one sequence, the 28 layers' heads in one view
        {"name": "keep 1x64", "op": "keep", "b": 1, "t": 64, "kv": 224, "dim": 128, "store": "bf16", "cap": 160},
        # the same for 32 sequences of an e4m3 cache
        {"name": "keep 32x16 e4m3", "op": "keep", "b": 32, "t": 16, "kv": 224, "dim": 128, "store": "e4m3", "cap": 96},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["cache", "attention", "attention", "verify", "keep"])
    dim = rng.choice([64, 128])
    if op == "cache":
        b = _log(rng, 1, 128)
        t = _log(rng, 1, max(1, min(2048, 32768 // b)))
        return {"op": op, "b": b, "t": t, "kv": rng.choice([1, 2, 3, 4, 5, 8]), "dim": dim, "store": rng.choice(["e4m3", "int8"]),
                "src": rng.choice(["bf16", "fp16", "fp32"]), "dst": rng.choice(["bf16", "fp16", "fp32"]), "cap": t + _log(rng, 1, 2048)}
    if op == "attention":
        b, t = _log(rng, 1, 128), _log(rng, 1, 64)
        kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        q = rng.choice(["bf16", "bf16", "fp16"])
        store, ragged = rng.choice([q, q, "e4m3", "int8"]), rng.random() < 0.7
        # at most the bytes of the serving case, and the arithmetic of the case with eight query heads for each K/V head
        most = min(8 * 128 * 8184 // (b * kv * SIZES[store]), 8 * 64 * 64 * 8128 // (b * t * kv * group))
        return {"op": op, "b": b, "t": t, "kv": kv, "group": group, "dim": dim, "q": q, "store": store,
                "len": _log(rng, 1, min(CAPACITY - t, most if ragged else most // 2)), "ragged": ragged, "shape": rng.choice(["chain", "tree"])}
    if op == "verify":
        vocab = rng.choice([VOCAB, VOCAB, _log(rng, 1000, VOCAB)])
        b = _log(rng, 1, 32)
        return {"op": op, "b": b, "t": _log(rng, 1, min(64, 256 // b)), "vocab": vocab, "type": rng.choice(["fp32", "fp32", "bf16"]),
                "draft": rng.random() < 0.5, "shape": rng.choice(["chain", "tree"]), "temp": rng.choice([0.0, 0.6, 1.0, 1.3])}
    b, t = _log(rng, 1, 32), _log(rng, 2, 64)
    return {"op": op, "b": b, "t": t, "kv": rng.choice([1, 8, 28, 56, 224]), "dim": dim, "store": rng.choice(["bf16", "fp16", "e4m3", "int8"]),
            "cap": t + _log(rng, 1, 64)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _parents(rng, b, t, shape, ragged):
    """Trees as drafters make them: a chain, or each node under one of the last few. Ragged batches end in absent nodes (-2)."""
    par = np.empty((b, t), np.int32)
    par[:, 0] = -1
    for i in range(1, t):
        par[:, i] = i - 1 if shape == "chain" else rng.randint(max(0, i - 6), i, b)
    if ragged:
        for s in range(b):
            if rng.rand() < 0.4:
                par[s, rng.randint(1, t + 1):] = -2
    return par


def _cache(g, b, kv, cap, dim, store):
    """A cache in the middle of its life. K rows have a few large channels, as trained models' have."""
    big = 1 + 7 * (torch.rand(1, kv, 1, dim, generator=g, device="cuda") < 0.03).float()
    out = {}
    for name in ("k", "v"):
        out[name] = torch.empty(b, kv, cap, dim, device="cuda", dtype=DTYPES[store])
        out[name + "_scale"] = torch.empty(b, kv, cap, device="cuda") if store in TOP else None
        for r in range(b):
            x = torch.randn(kv, cap, dim, generator=g, device="cuda")
            x = x * big[0] if name == "k" else x
            if store in TOP:
                scale = x.abs().amax(-1) / TOP[store]
                out[name + "_scale"][r] = scale
                x = x / scale[..., None]
            out[name][r] = (torch.round(x) if store == "int8" else x).to(DTYPES[store])
    return out


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    s = {"case": c}
    if c["op"] == "cache":
        shape = (c["b"], c["t"], c["kv"], c["dim"])
        s["kv"] = _cache(g, c["b"], c["kv"], c["cap"], c["dim"], c["store"])
        s["k"] = (torch.randn(shape, generator=g, device="cuda") * 3).to(DTYPES[c["src"]])
        s["v"] = torch.randn(shape, generator=g, device="cuda").to(DTYPES[c["src"]])
        s["start"] = torch.from_numpy(rng.randint(0, c["cap"] - c["t"] + 1, c["b"]).astype(np.int32)).cuda()
        counts = np.where(rng.rand(c["b"]) < 0.7, c["t"], rng.randint(0, c["t"] + 1, c["b"])) if c["t"] > 1 else np.ones(c["b"])
        counts[0] = c["t"]
        s["counts"] = torch.from_numpy(counts.astype(np.int32)).cuda()
        s["k_out"] = torch.zeros(shape, device="cuda", dtype=DTYPES[c["dst"]])
        s["v_out"] = torch.zeros(shape, device="cuda", dtype=DTYPES[c["dst"]])
    elif c["op"] == "attention":
        cap = c["len"] + c["t"]
        s["kv"] = _cache(g, c["b"], c["kv"], cap, c["dim"], c["store"])
        s["q"] = torch.randn(c["b"], c["t"], c["kv"] * c["group"], c["dim"], generator=g, device="cuda").to(DTYPES[c["q"]])
        s["out"] = torch.empty_like(s["q"])
        lens = np.full(c["b"], c["len"])
        if c["ragged"]:
            lens[1:] = rng.randint(0, c["len"] + 1, c["b"] - 1)
        s["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        s["parents"] = torch.from_numpy(_parents(rng, c["b"], c["t"], c["shape"], c["ragged"])).cuda()
        s["scale"] = 1.0 / math.sqrt(c["dim"])
    elif c["op"] == "verify":
        b, t, vocab = c["b"], c["t"], c["vocab"]
        par = _parents(rng, b, t, c["shape"], False)
        # the target's logits: a few likely tokens before a long tail; the drafter's are theirs, blurred
        logits = torch.randn(b, t, vocab, generator=g, device="cuda") * 3
        likely = torch.randint(0, vocab, (b, t, 8), generator=g, device="cuda")
        logits.scatter_(2, likely, 15 + 2 * torch.randn(b, t, 8, generator=g, device="cuda"))
        s["logits"] = logits.to(DTYPES[c["type"]])
        temp = c["temp"] or 1.0
        s["draft"] = torch.empty_like(logits) if c["draft"] else None
        tokens = torch.zeros(b, t, dtype=torch.int32, device="cuda")
        sibling = np.zeros((b, t), np.int64)
        for i in range(1, t):
            sibling[:, i] = (par[:, 1:i] == par[:, i:i + 1]).sum(1)
        for r in range(b):
            if c["draft"]:  # every child is drawn from its parent's row of the drafter's probabilities
                s["draft"][r] = torch.softmax((logits[r] + 0.7 * torch.randn(t, vocab, generator=g, device="cuda")) / temp, -1)
                picks = torch.multinomial(s["draft"][r], t, replacement=True, generator=g)
            else:  # the drafter's best guesses, one after another
                picks = torch.topk(logits[r] / temp - 0.8 * torch.log(-torch.log(torch.rand(t, vocab, generator=g, device="cuda").clamp(1e-6, 1 - 1e-6))), min(t, vocab), -1).indices
            at = torch.from_numpy(np.stack([np.maximum(par[r], 0), sibling[r]])).cuda().long()
            tokens[r, 1:] = picks[at[0, 1:], at[1, 1:]].int()
        s["tokens"] = tokens
        s["parents"] = torch.from_numpy(par).cuda()
        s["u"] = torch.rand(b, t, generator=g, device="cuda")
        s["path"] = torch.empty(b, t, dtype=torch.int32, device="cuda")
        s["n_path"] = torch.empty(b, dtype=torch.int32, device="cuda")
        s["next"] = torch.empty(b, dtype=torch.int32, device="cuda")
    else:
        s["kv"] = _cache(g, c["b"], c["kv"], c["cap"], c["dim"], c["store"])
        path, count = np.full((c["b"], c["t"]), -1, np.int32), np.empty(c["b"], np.int32)
        for r in range(c["b"]):
            n = min(c["t"], 1 + rng.randint(1, 8))
            path[r, :n] = np.concatenate([[0], 1 + np.sort(rng.choice(c["t"] - 1, n - 1, replace=False))])
            count[r] = n
        s["path"], s["n_path"] = torch.from_numpy(path).cuda(), torch.from_numpy(count).cuda()
        s["start"] = torch.from_numpy(rng.randint(0, c["cap"] - c["t"] + 1, c["b"]).astype(np.int32)).cuda()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"cache": _plain_cache, "attention": _plain_attention, "verify": _plain_verify, "keep": _plain_keep}[s["case"]["op"]](s)


def _view(s, qb):
    """The cache view that a program keeps beside its cache."""
    if "view" not in s:
        kv, c = s["kv"], s["case"]
        kind = {"bf16": qb.BF16, "fp16": qb.FP16, "e4m3": qb.E4M3, "int8": qb.INT8}[c["store"]]
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        s["view"] = qb.KVCache(ptr(kv["k"]), ptr(kv["v"]), ptr(kv["k_scale"]), ptr(kv["v_scale"]), kv["k"].stride(0), kv["k"].stride(1), kind,
                               kv["k"].shape[0], kv["k"].shape[1], c["dim"], kv["k"].shape[2])
    return s["view"]


def _own(s):
    qb, c = _library(), s["case"]
    kinds = {"bf16": qb.BF16, "fp16": qb.FP16, "fp32": qb.FP32}
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "cache":
        view, ld = _view(s, qb), c["kv"] * c["dim"]
        qb.kv_append(view, s["k"].data_ptr(), s["v"].data_ptr(), kinds[c["src"]], ld, c["t"], s["start"].data_ptr(), s["counts"].data_ptr(), stream)
        qb.kv_read(view, s["k_out"].data_ptr(), s["v_out"].data_ptr(), kinds[c["dst"]], ld, c["t"], s["start"].data_ptr(), s["counts"].data_ptr(), stream)
        return {"k": s["k_out"], "v": s["v_out"]}
    if c["op"] == "attention":
        view, heads = _view(s, qb), c["kv"] * c["group"]
        if "work" not in s:  # kept by the program, as large as the library asks for
            s["work"] = torch.empty(qb.tree_attention_workspace(view, c["t"], heads), dtype=torch.uint8, device="cuda")
        ld = heads * c["dim"]
        qb.tree_attention(view, s["q"].data_ptr(), s["out"].data_ptr(), kinds[c["q"]], ld, ld, c["t"], heads, s["lens"].data_ptr(),
                          s["parents"].data_ptr(), s["scale"], s["work"].data_ptr(), s["work"].numel(), stream)
        return {"out": s["out"]}
    if c["op"] == "verify":
        draft = s["draft"]
        qb.tree_verify(s["logits"].data_ptr(), kinds[c["type"]], c["vocab"], 0 if draft is None else draft.data_ptr(), c["vocab"], s["tokens"].data_ptr(),
                       s["parents"].data_ptr(), s["u"].data_ptr(), c["b"], c["t"], c["vocab"], c["temp"], s["path"].data_ptr(), s["n_path"].data_ptr(),
                       s["next"].data_ptr(), stream)
        return {"path": s["path"], "n_path": s["n_path"], "next": s["next"]}
    qb.kv_keep(_view(s, qb), s["start"].data_ptr(), s["path"].data_ptr(), s["n_path"].data_ptr(), c["t"], stream)
    return _whole(s["kv"])


def _whole(kv):
    return {n: x for n, x in kv.items() if x is not None}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_cache(s):
    c, kv = s["case"], s["kv"]
    t = torch.arange(c["t"], device="cuda")
    live = t[None] < s["counts"][:, None]                                                   # [b][t]
    at = (s["start"][:, None] + t[None]).long()
    seq = torch.arange(c["b"], device="cuda")[:, None].expand_as(at)
    out = {}
    for name in ("k", "v"):
        x = s[name].float()
        top = TOP[c["store"]]
        amax = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -60)
        y = x.double() * top / amax.double()                                                # 64 bits: next to a border the code depends on the last bit
        if c["store"] == "e4m3":
            step = torch.exp2((torch.frexp(y).exponent - 1).clamp_min(-6) - 3.0)            # between two neighbours of 3 mantissa bits
            code = (torch.round(y / step) * step).to(torch.float8_e4m3fn)
        else:
            code = torch.round(y).to(torch.int8)
        raw, scale = kv[name].view(torch.uint8), kv[name + "_scale"]
        raw[seq, :, at] = torch.where(live[:, :, None, None], code.view(torch.uint8), raw[seq, :, at])
        scale[seq, :, at] = torch.where(live[:, :, None], (amax / top)[..., 0], scale[seq, :, at])
        back = raw[seq, :, at].view(DTYPES[c["store"]]).float() * scale[seq, :, at][..., None]
        out[name] = torch.where(live[:, :, None, None], back.to(DTYPES[c["dst"]]), s[name + "_out"])
    return out


def _visible(parents, lens, cap):
    """[b][t][t]: whether node i sees node j (an ancestor of it, or itself); absent nodes see nothing."""
    b, t = parents.shape
    i = torch.arange(t, device=parents.device)
    fine = (parents >= -1) & (parents < i) & (lens[:, None] >= 0) & (lens[:, None] + i < cap)
    step = (parents[:, :, None] == i) & fine[:, :, None]
    reach = torch.linalg.matrix_power(step.float() + torch.eye(t, device=parents.device), max(1, t - 1)) > 0
    present = ~(reach & ~fine[:, None, :]).any(-1)
    return reach & present[:, :, None]


def _plain_attention(s):
    c, kv = s["case"], s["kv"]
    b, t, h, n, d = c["b"], c["t"], c["kv"], c["group"], c["dim"]
    k, v = kv["k"].float(), kv["v"].float()
    if kv["k_scale"] is not None:
        k, v = k * kv["k_scale"][..., None], v * kv["v_scale"][..., None]
    cap = k.shape[2]
    q = s["q"].float().view(b, t, h, n, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * n, d)
    score = q @ k.transpose(-1, -2) * s["scale"]
    del k
    sees = _visible(s["parents"], s["lens"], cap)                                           # [b][t][t]
    pos = torch.arange(cap, device="cuda")
    node = pos - s["lens"][:, None]                                                         # [b][cap]
    branch = torch.gather(sees, 2, node.clamp(0, t - 1)[:, None].expand(b, t, cap)) & (node >= 0)[:, None] & (node < t)[:, None]
    mask = branch | ((node < 0)[:, None] & sees.any(-1)[..., None])                         # [b][t][cap]
    mask = mask[:, None, :, None].expand(b, 1, t, n, cap).reshape(b, 1, t * n, cap)
    score = score.masked_fill_(~mask, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return {"out": o.view(b, h, t, n, d).permute(0, 2, 1, 3, 4).reshape(b, t, h * n, d).to(DTYPES[c["q"]])}


def _plain_verify(s):
    """Parents come before their children, so one pass over the nodes in order is the walk: `at` is the node that it has reached,
    p the target's probabilities there, r what is left of them after the refused children, left its sum."""
    c = s["case"]
    b, t = c["b"], c["t"]
    seq = torch.arange(b, device="cuda")
    at = torch.zeros(b, dtype=torch.int64, device="cuda")
    reached = torch.zeros(b, t, dtype=torch.bool, device="cuda")
    reached[:, 0] = True

    def probabilities(node):
        x = s["logits"][seq, node].double()
        if c["temp"] == 0:
            return torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
        p = ((x - x.amax(1, keepdim=True)) / c["temp"]).exp()
        return p / p.sum(1, keepdim=True)

    p = r = probabilities(at)
    left = torch.ones(b, dtype=torch.float64, device="cuda")
    share = torch.zeros_like(left)                                                          # how often q has been taken from p
    for i in range(1, t):
        tried = s["parents"][:, i].long() == at
        x, u = s["tokens"][:, i].long()[:, None], s["u"][:, i].double()
        if s["draft"] is not None and c["temp"] > 0:
            q = s["draft"][seq, at].double()
            take = tried & (u * left * q.gather(1, x)[:, 0] < r.gather(1, x)[:, 0])
            rest = (p - (share + left)[:, None] * q).clamp_min(0)
        else:
            take = tried & (u * left < r.gather(1, x)[:, 0])
            rest = r.scatter(1, x, 0.0)
        refused = tried & ~take
        share = torch.where(refused, share + left, share)
        r = torch.where(refused[:, None], rest, r)
        left = torch.where(refused, rest.sum(1), left)
        at = torch.where(take, i, at)
        reached[:, i] = take
        p = torch.where(take[:, None], probabilities(at), p)
        r = torch.where(take[:, None], p, r)
        left, share = torch.where(take, 1.0, left), torch.where(take, 0.0, share)
    r = torch.where((left > 0)[:, None], r, p)
    sums = r.cumsum(1)
    token = (sums > (s["u"][:, 0].double() * sums[:, -1])[:, None]).long().argmax(1)
    order = torch.where(reached, torch.arange(t, device="cuda"), t).sort(1).values
    return {"path": torch.where(order < t, order, -1).int(), "n_path": reached.sum(1).int(), "next": token.int()}


def _plain_keep(s):
    c, kv = s["case"], s["kv"]
    i = torch.arange(c["t"], device="cuda")
    live = i[None] < s["n_path"][:, None]
    src = (s["start"][:, None] + torch.where(live, s["path"], i.int()[None])).long()
    dst = (s["start"][:, None] + i[None]).long()
    seq = torch.arange(c["b"], device="cuda")[:, None].expand_as(dst)
    for x in _whole(kv).values():
        raw = x.view(torch.uint8) if c["store"] in TOP and x.dim() == 4 else x
        raw[seq, :, dst] = raw[seq, :, src]
    return _whole(kv)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "cache":
        rows = c["b"] * c["t"] * c["kv"] * 2
        rows *= 1.0 if c["t"] == 1 else 0.85                                                # 30 % of the sequences bring half of their rows
        return {"bytes": rows * (c["dim"] * (SIZES[c["src"]] + 2 + SIZES[c["dst"]]) + 8), "flops": rows * c["dim"] * 4.0}
    if c["op"] == "attention":
        positions = c["b"] * (c["len"] * (0.5 if c["ragged"] and c["b"] > 1 else 1.0) + c["t"])
        row = c["dim"] * SIZES[c["store"]] + (4 if c["store"] in TOP else 0)
        heads = c["kv"] * c["group"]
        return {"bytes": positions * c["kv"] * 2 * row + c["b"] * c["t"] * heads * c["dim"] * 2 * SIZES[c["q"]],
                "flops": 4.0 * positions * c["t"] * heads * c["dim"]}
    if c["op"] == "verify":
        # the rows of the nodes that the walk reaches (about three of four drafted tokens are kept), and the last one's drafted probabilities
        levels = c["t"] if c["shape"] == "chain" else min(c["t"], 2 + int(math.log2(c["t"])))
        rows = sum(0.73 ** k for k in range(levels)) if c["temp"] > 0 else 1.0 + (levels > 1) * 0.5
        drafted = 1.0 if c["draft"] and c["temp"] > 0 and c["t"] > 1 else 0.0
        return {"bytes": c["b"] * c["vocab"] * (rows * SIZES[c["type"]] + 4.0 * drafted), "flops": c["b"] * c["vocab"] * 4.0 * (rows + drafted)}
    moved = c["b"] * c["kv"] * 2 * min(c["t"] - 1, 4)                                       # about four accepted rows beside the first
    return {"bytes": 2.0 * moved * (c["dim"] * SIZES[c["store"]] + (4 if c["store"] in TOP else 0)), "flops": 0.0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _e4m3(y):
    """The nearest of the type's finite values (ties to the even code), from the list of them."""
    code = torch.arange(127, device=y.device)
    e, m = code >> 3, (code & 7).double()
    values = torch.where(e == 0, m / 512, (1 + m / 8) * torch.exp2(e - 7.0))
    x = y.abs().clamp_max(448.0)
    up = torch.searchsorted(values, x).clamp_max(126)                                       # the first value >= x
    down = (up - 1).clamp_min(0)
    a, b = x - values[down], values[up] - x
    return torch.where((a < b) | ((a == b) & (down % 2 == 0)), values[down], values[up]) * y.sign()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "cache":
        out = {}
        for name in ("k", "v"):
            x = s[name].double()
            whole = torch.zeros_like(x)
            for r, n in enumerate(s["counts"].tolist()):
                row = x[r, :n]
                amax = row.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -60)
                y = row * TOP[c["store"]] / amax
                whole[r, :n] = (torch.round(y) if c["store"] == "int8" else _e4m3(y)) * amax / TOP[c["store"]]
            out[name] = whole
        return out
    if c["op"] == "attention":
        b, t, h, n = c["b"], c["t"], c["kv"], c["group"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        parents, lens = s["parents"].tolist(), s["lens"].tolist()
        for r in range(b):
            length = lens[r]
            sets = []
            for i in range(t):
                up, j = [], i
                while j >= 0:
                    up.append(j)
                    j = parents[r][j]
                sets.append(up if j == -1 else None)
            k, v = s["kv"]["k"][r, :, :length + t].double(), s["kv"]["v"][r, :, :length + t].double()
            if s["kv"]["k_scale"] is not None:
                k = k * s["kv"]["k_scale"][r, :, :length + t, None].double()
                v = v * s["kv"]["v_scale"][r, :, :length + t, None].double()
            allowed = torch.zeros(t, length + t, dtype=torch.bool)
            for i, up in enumerate(sets):
                if up is not None:
                    allowed[i, :length] = True
                    allowed[i, [length + j for j in up]] = True
            allowed = allowed.cuda()
            rows = allowed.any(1).nonzero()[:, 0]
            if not len(rows):
                continue
            q = s["q"][r].double().view(t, h, n, c["dim"])[rows]
            w = torch.einsum("thnd,hkd->hntk", q, k) * s["scale"]
            w = torch.softmax(w.masked_fill(~allowed[rows], -math.inf), -1)
            out[r, rows] = torch.einsum("hntk,hkd->thnd", w, v).reshape(len(rows), h * n, c["dim"])
        return {"out": out}
    if c["op"] == "verify":
        paths, counts, ends = [], [], []
        parents, tokens, u = s["parents"].tolist(), s["tokens"].tolist(), s["u"].double().tolist()
        for r in range(c["b"]):
            at, path, searching = 0, [0], True
            while searching:
                searching = False
                x = s["logits"][r, at].double().cpu().numpy()
                if c["temp"] == 0:
                    p = np.zeros_like(x)
                    p[int(np.argmax(x))] = 1.0
                else:
                    p = np.exp((x - x.max()) / c["temp"])
                    p /= p.sum()
                rest = p.copy()
                q = s["draft"][r, at].double().cpu().numpy() if s["draft"] is not None and c["temp"] > 0 else None
                for i in range(at + 1, c["t"]):
                    if parents[r][i] != at:
                        continue
                    x, total = tokens[r][i], rest.sum()
                    if u[r][i] * total * (1.0 if q is None else q[x]) < rest[x]:
                        at, searching = i, True
                        path.append(i)
                        break
                    if q is None:
                        rest[x] = 0.0
                    else:
                        rest = np.maximum(rest - total * q, 0.0)
            sums = np.cumsum(rest if rest.sum() > 0 else p)
            ends.append(int(np.argmax(sums > u[r][0] * sums[-1])))
            paths.append(path + [-1] * (c["t"] - len(path)))
            counts.append(len(path))
        return {"path": np.array(paths, np.int32), "n_path": np.array(counts, np.int32), "next": np.array(ends, np.int32)}
    kv = {n: x.float().double() for n, x in _whole(s["kv"]).items()}
    for x in kv.values():
        for r, (start, n) in enumerate(zip(s["start"].tolist(), s["n_path"].tolist())):
            x[r, :, start:start + n] = x[r][:, [start + j for j in s["path"][r, :n].tolist()]].clone()
    return kv
