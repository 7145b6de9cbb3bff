"""Cases and plain forms of the operators of serving over a K/V cache in pages.

Four operators, one pass of each:
  rope       the heads' norms and the position rotation of new Q and K rows; K and V go to their pages
  prompt     causal attention of whole prompts of different lengths, packed one behind the other
  paged      attention of one new token a sequence over its pages
  logprobs   log probabilities of given tokens, entropies and the likeliest alternatives

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
BASE = 1e6           # the model's rotation base
EPS = 1e-6
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
        # one decode step of a full batch: a token's rows per sequence into bf16 pages
        {"name": "rope step 128", "op": "rope", "b": 128, "rows": 1, "heads": 16, "kv": 8, "dim": 128, "src": "bf16", "out": "bf16", "store": "bf16", "page": 16, "keys": False},
        # four prompts of 2048 tokens entering pages; K goes on to the prompts' attention too
        {"name": "rope prompts 4x2048", "op": "rope", "b": 4, "rows": 2048, "heads": 16, "kv": 8, "dim": 128, "src": "bf16", "out": "bf16", "store": "bf16", "page": 64, "keys": True},
        # odd sizes, fp32 projections, heads of 64
        {"name": "rope odd fp32", "op": "rope", "b": 3, "rows": 517, "heads": 15, "kv": 5, "dim": 64, "src": "fp32", "out": "fp16", "store": "fp16", "page": 32, "keys": True},
        # one short question
        {"name": "prompt 1x100", "op": "prompt", "b": 1, "len": 100, "context": 0, "heads": 16, "kv": 8, "dim": 128, "type": "bf16", "ragged": False},
        # a serving batch: parts of prompts behind contexts of up to 1000 tokens, heads of 64
        {"name": "prompt 16 ragged fp16", "op": "prompt", "b": 16, "len": 1900, "context": 1000, "heads": 12, "kv": 4, "dim": 64, "type": "fp16", "ragged": True},
        # a prompt as long as a cache slot
        {"name": "prompt 1x8192", "op": "prompt", "b": 1, "len": 8192, "context": 0, "heads": 16, "kv": 8, "dim": 128, "type": "bf16", "ragged": False},
        # one sequence: the latency of plain decoding
        {"name": "paged 1 at 1024", "op": "paged", "b": 1, "heads": 16, "kv": 8, "dim": 128, "q": "bf16", "store": "bf16", "page": 16, "len": 1024, "ragged": False},
        # a batch over ragged int8 pages, heads of 64, seven query heads each
        {"name": "paged 32 int8", "op": "paged", "b": 32, "heads": 28, "kv": 4, "dim": 64, "q": "fp16", "store": "int8", "page": 32, "len": 4099, "ragged": True},
        # serving: 128 sequences over ragged e4m3 pages
        {"name": "paged 128 e4m3", "op": "paged", "b": 128, "heads": 16, "kv": 8, "dim": 128, "q": "bf16", "store": "e4m3", "page": 64, "len": 8191, "ragged": True},
        # the token just sampled, as an interface that returns alternatives asks for it
        {"name": "logprobs 1 top 20", "op": "logprobs", "rows": 1, "vocab": VOCAB, "type": "fp32", "temp": 1.0, "top": 20},
        # a batch's step
        {"name": "logprobs 128 top 5", "op": "logprobs", "rows": 128, "vocab": VOCAB, "type": "fp32", "temp": 0.6, "top": 5},
        # scoring a prompt of 2048 tokens
        {"name": "logprobs 2048 bf16", "op": "logprobs", "rows": 2048, "vocab": VOCAB, "type": "bf16", "temp": 1.0, "top": 1},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "prompt", "paged", "paged", "logprobs"])
    dim = rng.choice([64, 128])
    if op == "rope":
        b = _log(rng, 1, 128)
        kv = rng.choice([1, 2, 4, 5, 8])
        src = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": op, "b": b, "rows": _log(rng, 1, max(1, min(2048, 8192 // b) * (1 if src != "fp32" else 2) // 2)), "heads": kv * rng.choice([1, 2, 3]), "kv": kv, "dim": dim,
                "src": src, "out": rng.choice(["bf16", "fp16"]), "store": rng.choice(["bf16", "fp16"]), "page": rng.choice([8, 16, 32, 64, 128]), "keys": rng.random() < 0.5}
    if op == "prompt":
        kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        b, context = _log(rng, 1, 16), rng.choice([0, 0, 1]) * _log(rng, 1, 4096)
        most = 16 * 8192 * 8192 // 2 // (b * kv * group)                                    # products as the prompt of 8192 has
        longest = int(math.sqrt(context * context + 2 * most) - context)
        return {"op": op, "b": b, "len": _log(rng, 1, max(1, min(8192, longest, 32768 // b))), "context": context, "heads": kv * group, "kv": kv, "dim": dim,
                "type": rng.choice(["bf16", "bf16", "fp16"]), "ragged": rng.random() < 0.7}
    if op == "paged":
        b, kv, group = _log(rng, 1, 128), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        q = rng.choice(["bf16", "bf16", "fp16"])
        store, ragged = rng.choice([q, q, "e4m3", "int8"]), rng.random() < 0.7
        most = 128 * 8 * 8191 * 128 // (b * kv * SIZES[store] * dim)                        # bytes as the serving batch has
        return {"op": op, "b": b, "heads": kv * group, "kv": kv, "dim": dim, "q": q, "store": store, "page": rng.choice([8, 16, 32, 64, 128]),
                "len": _log(rng, 1, min(32767, most if ragged else most // 2)), "ragged": ragged}
    vocab = rng.choice([VOCAB, VOCAB, _log(rng, 1000, VOCAB)])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    return {"op": op, "rows": _log(rng, 1, 2048 * 2 // SIZES[kind]), "vocab": vocab, "type": kind, "temp": rng.choice([0.6, 1.0, 1.3]), "top": rng.choice([0, 1, 5, 20, 64])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _sizes(c):
    """Rows and contexts of a case's sequences, the same for every seed: the outputs' shapes hang on them."""
    rng, b = np.random.RandomState(c["b"] * 7919 + c.get("rows", c.get("len"))), c["b"]
    if c["op"] == "rope":    # one token each, or prompts of up to `rows` tokens
        count = np.ones(b, np.int64) if c["rows"] == 1 else np.where(rng.rand(b) < 0.5, c["rows"], rng.randint(1, c["rows"] + 1, b))
        count[0] = c["rows"]
        return count, None
    lens, context = np.full(b, c["len"]), np.full(b, c.get("context", 0))
    if c["ragged"]:
        lens[1:] = rng.randint(0 if c["op"] == "paged" else 1, c["len"] + 1, b - 1)
        context[1:] = rng.randint(0, c.get("context", 0) + 1, b - 1)
    return lens, context


def _tables(rng, needed, page, first=None):
    """Page numbers of sequences that hold positions first .. needed - 1, in the order in which a pool gives pages out; pages
    before the first are given back (-1)."""
    low = np.zeros(len(needed), np.int64) if first is None else first // page
    high = (np.asarray(needed, np.int64) + page - 1) // page
    table = np.full((len(needed), int(high.max()) + 1), -1, np.int32)
    spare = 3 if first is None else 3 + int((-(-(np.asarray(needed) - first) // page) + 1 - (high - low)).sum())   # (as many pages for every seed)
    pool = rng.permutation(int((high - low).sum()) + spare).astype(np.int32)
    at = 0
    for r in range(len(needed)):
        n = int(high[r] - low[r])
        table[r, low[r]:high[r]] = pool[at:at + n]
        at += n
    return table, len(pool)


def _pool(g, pages, kv, page, dim, store):
    """A pool of pages in the middle of its life. K rows have a few large channels, as trained models' have."""
    big = 1 + 7 * (torch.rand(1, kv, 1, dim, generator=g, device="cuda") < 0.03).float()
    out = {}
    for name in ("k", "v"):
        out[name] = torch.empty(pages, kv, page, dim, device="cuda", dtype=DTYPES[store])
        out[name + "_scale"] = torch.empty(pages, kv, page, device="cuda") if store in TOP else None
        step = max(1, (1 << 26) // (kv * page * dim))
        for p in range(0, pages, step):
            x = torch.randn(min(step, pages - p), kv, page, dim, generator=g, device="cuda")
            x = x * big if name == "k" else x
            if store in TOP:
                scale = x.abs().amax(-1) / TOP[store]
                out[name + "_scale"][p:p + step] = scale
                x = x / scale[..., None]
            out[name][p:p + step] = (torch.round(x) if store == "int8" else x).to(DTYPES[store])
    return out


def _dev(a, kind=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a).astype(kind)).cuda()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    s = {"case": c}
    if c["op"] == "rope":
        count, _ = _sizes(c)                                                                # behind contexts whose oldest pages were given back
        first = rng.randint(0, 32768, c["b"])
        first[0] = 0 if c["rows"] > 1 else first[0]
        n = int(count.sum())
        table, pages = _tables(rng, first + count, c["page"], first)
        s["kv"] = _pool(g, pages, c["kv"], c["page"], c["dim"], c["store"])
        s["table"] = _dev(table)
        s["seqs"] = _dev(np.repeat(np.arange(c["b"]), count))
        s["positions"] = _dev(np.concatenate([np.arange(a, a + m) for a, m in zip(first, count)]))
        for name, heads in (("q", c["heads"]), ("k", c["kv"]), ("v", c["kv"])):
            s[name] = (torch.randn(n, heads * c["dim"], generator=g, device="cuda") * 2).to(DTYPES[c["src"]])
        for name in ("q_gain", "k_gain"):
            s[name] = (1 + 0.3 * torch.randn(c["dim"], generator=g, device="cuda")).bfloat16()
        s["q_out"] = torch.empty(n, c["heads"] * c["dim"], device="cuda", dtype=DTYPES[c["out"]])
        s["k_out"] = torch.empty(n, c["kv"] * c["dim"], device="cuda", dtype=DTYPES[c["out"]]) if c["keys"] else None
    elif c["op"] == "prompt":
        lens, context = _sizes(c)
        s["lens"], s["context"] = lens.tolist(), context.tolist()
        s["starts"], s["k_starts"] = _dev(np.concatenate([[0], np.cumsum(lens)])), _dev(np.concatenate([[0], np.cumsum(lens + context)]))
        n, m = int(lens.sum()), int((lens + context).sum())
        s["q"] = torch.randn(n, c["heads"] * c["dim"], generator=g, device="cuda").to(DTYPES[c["type"]])
        s["k"] = torch.randn(m, c["kv"] * c["dim"], generator=g, device="cuda").to(DTYPES[c["type"]])
        s["v"] = torch.randn(m, c["kv"] * c["dim"], generator=g, device="cuda").to(DTYPES[c["type"]])
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(c["dim"])
    elif c["op"] == "paged":
        lens, _ = _sizes(c)
        table, pages = _tables(rng, lens + 1, c["page"])
        s["kv"] = _pool(g, pages, c["kv"], c["page"], c["dim"], c["store"])
        s["table"], s["lens"] = _dev(table), _dev(lens)
        s["q"] = torch.randn(c["b"], c["heads"] * c["dim"], generator=g, device="cuda").to(DTYPES[c["q"]])
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(c["dim"])
    else:
        # a few likely tokens before a long tail; the given token is often one of them
        n, vocab = c["rows"], c["vocab"]
        likely = torch.randint(0, vocab, (n, 8), generator=g, device="cuda")
        values = 15 + 2 * torch.randn(n, 8, generator=g, device="cuda")
        s["logits"] = torch.empty(n, vocab, device="cuda", dtype=DTYPES[c["type"]])
        for r in range(0, n, 256):
            x = torch.randn(min(256, n - r), vocab, generator=g, device="cuda") * 3
            s["logits"][r:r + 256] = x.scatter_(1, likely[r:r + 256], values[r:r + 256]).to(DTYPES[c["type"]])
        other = torch.randint(0, vocab, (n,), generator=g, device="cuda")
        s["tokens"] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.8, likely[:, 0], other).int()
        s["logprob"], s["entropy"] = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        s["top_ids"] = torch.empty(n, c["top"], device="cuda", dtype=torch.int32)
        s["top_logprobs"] = torch.empty(n, c["top"], device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "prompt": _plain_prompt, "paged": _plain_paged, "logprobs": _plain_logprobs}[s["case"]["op"]](s)


def _view(s, qb):
    """The view of the pages that a program keeps beside its pool."""
    if "view" not in s:
        kv, c = s["kv"], s["case"]
        kind = {"bf16": qb.BF16, "fp16": qb.FP16, "e4m3": qb.E4M3, "int8": qb.INT8}[c["store"]]
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        s["view"] = qb.KVPages(ptr(kv["k"]), ptr(kv["v"]), ptr(kv["k_scale"]), ptr(kv["v_scale"]), s["table"].data_ptr(), kv["k"].stride(0), kv["k"].stride(1),
                               kind, kv["k"].shape[0], s["table"].shape[0], c["kv"], c["dim"], c["page"], s["table"].shape[1])
    return s["view"]


def _own(s):
    qb, c = _library(), s["case"]
    kinds = {"bf16": qb.BF16, "fp16": qb.FP16, "fp32": qb.FP32}
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "rope":
        wide, narrow = c["heads"] * c["dim"], c["kv"] * c["dim"]
        qb.qk_rope(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), kinds[c["src"]], wide, narrow, narrow, s["q"].shape[0], c["heads"], c["kv"], c["dim"],
                   s["q_gain"].data_ptr(), s["k_gain"].data_ptr(), qb.BF16, EPS, BASE, s["positions"].data_ptr(), s["q_out"].data_ptr(),
                   s["k_out"].data_ptr() if c["keys"] else 0, kinds[c["out"]], wide, narrow, _view(s, qb), s["seqs"].data_ptr(), stream)
        return _whole({"q_out": s["q_out"], "k_out": s["k_out"], **s["kv"]})
    if c["op"] == "prompt":
        wide, narrow = c["heads"] * c["dim"], c["kv"] * c["dim"]
        qb.prompt_attention(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), kinds[c["type"]], wide, narrow, narrow, wide,
                            s["starts"].data_ptr(), s["k_starts"].data_ptr(), c["b"], s["q"].shape[0], s["k"].shape[0], c["heads"], c["kv"], c["dim"], s["scale"], stream)
        return {"out": s["out"]}
    if c["op"] == "paged":
        view, wide = _view(s, qb), c["heads"] * c["dim"]
        if "work" not in s:  # kept by the program, as large as the library asks for
            s["work"] = torch.empty(qb.paged_attention_workspace(view, c["heads"]), dtype=torch.uint8, device="cuda")
        qb.paged_attention(view, s["q"].data_ptr(), s["out"].data_ptr(), kinds[c["q"]], wide, wide, c["heads"], s["lens"].data_ptr(), s["scale"],
                           s["work"].data_ptr(), s["work"].numel(), stream)
        return {"out": s["out"]}
    qb.token_logprobs(s["logits"].data_ptr(), kinds[c["type"]], c["vocab"], c["rows"], c["vocab"], s["tokens"].data_ptr(), c["temp"], c["top"],
                      s["logprob"].data_ptr(), s["entropy"].data_ptr(), s["top_ids"].data_ptr() if c["top"] else 0,
                      s["top_logprobs"].data_ptr() if c["top"] else 0, stream)
    return {n: s[n] for n in ("logprob", "entropy", "top_ids", "top_logprobs") if c["top"] or not n.startswith("top")}


def _whole(kv):
    return {n: x for n, x in kv.items() if x is not None}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_rope(s):
    c, kv = s["case"], s["kv"]
    half = c["dim"] // 2
    # 64 bits: a far position's angle needs more than 24
    angle = s["positions"].double()[:, None] * BASE ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    rows = {}
    for name, heads in (("q", c["heads"]), ("k", c["kv"])):
        x = s[name].float().view(-1, heads, c["dim"])
        x = x / (x * x).mean(-1, keepdim=True).add(EPS).sqrt() * s[name + "_gain"].float()
        a, b = x[..., :half], x[..., half:]
        rows[name] = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    rows["v"] = s["v"].float().view(-1, c["kv"], c["dim"])
    s["q_out"].copy_(rows["q"].view(s["q_out"].shape))
    if c["keys"]:
        s["k_out"].copy_(rows["k"].view(s["k_out"].shape))
    at = s["positions"].long()
    page = s["table"][s["seqs"].long(), at // c["page"]].long()
    for name in ("k", "v"):
        kv[name][page, :, at % c["page"]] = rows[name].to(DTYPES[c["store"]])
    return _whole({"q_out": s["q_out"], "k_out": s["k_out"], **kv})


def _plain_prompt(s):
    c = s["case"]
    group, d = c["heads"] // c["kv"], c["dim"]
    out, r0, k0 = [], 0, 0
    for n, context in zip(s["lens"], s["context"]):
        m = n + context
        q = s["q"][r0:r0 + n].float().view(n, c["kv"], group, d).permute(1, 2, 0, 3)
        k = s["k"][k0:k0 + m].float().view(m, c["kv"], 1, d).permute(1, 2, 0, 3)
        v = s["v"][k0:k0 + m].float().view(m, c["kv"], 1, d).permute(1, 2, 0, 3)
        score = q @ k.transpose(-1, -2) * s["scale"]
        later = torch.arange(m, device="cuda") > torch.arange(n, device="cuda")[:, None] + context
        score.masked_fill_(later, -math.inf)
        p = score.sub_(score.amax(-1, keepdim=True)).exp_()
        o = (p @ v) / p.sum(-1, keepdim=True)
        out.append(o.permute(2, 0, 1, 3).reshape(n, c["heads"] * d))
        r0, k0 = r0 + n, k0 + m
    return {"out": torch.cat(out).to(DTYPES[c["type"]])}


def _plain_paged(s):
    c, kv = s["case"], s["kv"]
    b, h, n, d = c["b"], c["kv"], c["heads"] // c["kv"], c["dim"]
    table = s["table"].long().clamp_min(0)

    def gathered(name):
        x = kv[name][table].float()                                                         # [b][pages][heads][page][dim]
        if kv[name + "_scale"] is not None:
            x = x * kv[name + "_scale"][table][..., None]
        return x.transpose(1, 2).reshape(b, h, -1, d)

    q = s["q"].float().view(b, h, n, d)
    score = q @ gathered("k").transpose(-1, -2) * s["scale"]
    hidden = torch.arange(score.shape[-1], device="cuda") > s["lens"][:, None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = (p @ gathered("v")) / p.sum(-1, keepdim=True)
    return {"out": o.reshape(b, c["heads"] * d).to(DTYPES[c["q"]])}


def _plain_logprobs(s):
    c = s["case"]
    back = torch.arange(c["vocab"], device="cuda").neg().add_(c["vocab"])
    for r in range(0, c["rows"], 256):
        raw = s["logits"][r:r + 256].float()
        x = (raw / c["temp"]).double()                                                      # 64 bits: long sums
        x = x - x.amax(1, keepdim=True)
        p = x.exp()
        total = p.sum(1, keepdim=True)
        x = x - total.log()
        s["logprob"][r:r + 256] = x.gather(1, s["tokens"][r:r + 256].long()[:, None])[:, 0]
        s["entropy"][r:r + 256] = -(p / total * x).sum(1)
        if c["top"]:
            # larger logits first, equal ones by their index: whole numbers in that order
            bits = torch.where(raw == 0, 0.0, raw).view(torch.int32)
            key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32) + back
            ids = key.topk(c["top"], 1).indices
            s["top_ids"][r:r + 256] = ids
            s["top_logprobs"][r:r + 256] = x.gather(1, ids)
    return {n: s[n] for n in ("logprob", "entropy", "top_ids", "top_logprobs") if c["top"] or not n.startswith("top")}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "rope":
        n = int(_sizes(c)[0].sum())
        into, out, store = SIZES[c["src"]], SIZES[c["out"]], SIZES[c["store"]]
        elems = c["heads"] * (into + out) + c["kv"] * (2 * into + 2 * store + (out if c["keys"] else 0))
        return {"bytes": n * (c["dim"] * elems + 8), "flops": n * (c["heads"] + c["kv"]) * c["dim"] * 8.0}
    if c["op"] == "prompt":
        lens, context = _sizes(c)
        n, m = int(lens.sum()), int((lens + context).sum())
        total = int((lens * (lens + 1) // 2 + lens * context).sum())                        # pairs of a query and a key that it sees
        return {"bytes": (2 * n * c["heads"] + 2 * m * c["kv"]) * c["dim"] * SIZES[c["type"]], "flops": 4.0 * total * c["heads"] * c["dim"]}
    if c["op"] == "paged":
        positions = int((_sizes(c)[0] + 1).sum())
        row = c["dim"] * SIZES[c["store"]] + (4 if c["store"] in TOP else 0)
        return {"bytes": positions * c["kv"] * 2 * row + c["b"] * c["heads"] * c["dim"] * 2 * SIZES[c["q"]], "flops": 4.0 * positions * c["heads"] * c["dim"]}
    n = float(c["rows"] * c["vocab"])
    return {"bytes": n * SIZES[c["type"]] + c["rows"] * (12 + 8 * c["top"]), "flops": n * 6.0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        d, out = c["dim"], {}
        rows = {"v": s["v"].double().view(-1, c["kv"], d)}
        positions = s["positions"].double()
        for name in ("q", "k"):
            x = s[name].double().view(s[name].shape[0], -1, d)
            x = x * torch.rsqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * s[name + "_gain"].double()
            turned = torch.empty_like(x)
            for j in range(d // 2):
                angle = positions * math.pow(BASE, -2.0 * j / d)
                co, si = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
                turned[..., j] = x[..., j] * co - x[..., j + d // 2] * si
                turned[..., j + d // 2] = x[..., j] * si + x[..., j + d // 2] * co
            rows[name] = turned
        out["q_out"] = rows["q"].reshape(s["q_out"].shape)
        if c["keys"]:
            out["k_out"] = rows["k"].reshape(s["k_out"].shape)
        table, seqs, at = s["table"].cpu().numpy(), s["seqs"].cpu().numpy(), s["positions"].cpu().numpy()
        row = torch.from_numpy(table[seqs, at // c["page"]].astype(np.int64) * c["page"] + at % c["page"]).cuda()
        for name in ("k", "v"):
            whole = s["kv"][name].double().transpose(1, 2).reshape(-1, c["kv"], d)
            whole.index_copy_(0, row, rows[name])
            out[name] = whole.view(-1, c["page"], c["kv"], d).transpose(1, 2)
        return out
    if c["op"] == "prompt":
        group, d = c["heads"] // c["kv"], c["dim"]
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        starts, k_starts = s["starts"].tolist(), s["k_starts"].tolist()
        for r in range(c["b"]):
            rows, keys = range(starts[r], starts[r + 1]), slice(k_starts[r], k_starts[r + 1])
            ahead = (k_starts[r + 1] - k_starts[r]) - len(rows)
            for h in range(c["heads"]):
                k = s["k"][keys, h // group * d:(h // group + 1) * d].double()
                v = s["v"][keys, h // group * d:(h // group + 1) * d].double()
                for i in range(0, len(rows), 2048):
                    part = slice(rows.start + i, min(rows.start + i + 2048, rows.stop))
                    w = s["q"][part, h * d:(h + 1) * d].double() @ k.T * s["scale"]
                    seen = torch.ones_like(w, dtype=torch.bool).tril(ahead + i)
                    out[part, h * d:(h + 1) * d] = torch.softmax(torch.where(seen, w, -math.inf), -1) @ v
        return {"out": out}
    if c["op"] == "paged":
        group, d = c["heads"] // c["kv"], c["dim"]
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for r, length in enumerate(s["lens"].tolist()):
            pages = s["table"][r, :length // c["page"] + 1].long()
            k, v = (s["kv"][n][pages].double().transpose(0, 1).reshape(c["kv"], -1, d)[:, :length + 1] for n in ("k", "v"))
            if s["kv"]["k_scale"] is not None:
                k, v = (x * s["kv"][n][pages].double().transpose(0, 1).reshape(c["kv"], -1, 1)[:, :length + 1] for x, n in ((k, "k_scale"), (v, "v_scale")))
            w = torch.softmax(torch.einsum("hgd,hkd->hgk", s["q"][r].double().view(c["kv"], group, d), k) * s["scale"], -1)
            out[r] = torch.einsum("hgk,hkd->hgd", w, v).reshape(-1)
        return {"out": out}
    logprob, entropy, ids, likely = [], [], [], []
    for r in range(c["rows"]):
        raw = s["logits"][r].double()
        y = raw / c["temp"]
        y = y - torch.logsumexp(y, 0)
        logprob.append(y[int(s["tokens"][r])])
        entropy.append(-(y.exp() * y).sum())
        best = torch.sort(raw, descending=True, stable=True).indices[:c["top"]]
        ids.append(best)
        likely.append(y[best])
    out = {"logprob": torch.stack(logprob), "entropy": torch.stack(entropy)}
    if c["top"]:
        out["top_ids"], out["top_logprobs"] = torch.stack(ids).int(), torch.stack(likely)
    return out
