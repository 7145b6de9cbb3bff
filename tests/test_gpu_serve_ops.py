"""The operators of serving over a K/V cache in pages (qwen_qk_rope, qwen_prompt_attention,
qwen_paged_attention, qwen_token_logprobs) against plain implementations in 64 bits, within
the roundings that their documentation names."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOP = {"e4m3": 448.0, "int8": 127.0}
DIRTY = 0x5A      # what unwritten bytes of pools and outputs hold


def _types(qb):
    import torch
    return {"bf16": (qb.BF16, torch.bfloat16), "fp16": (qb.FP16, torch.float16), "fp32": (qb.FP32, torch.float32),
            "e4m3": (qb.E4M3, torch.float8_e4m3fn), "int8": (qb.INT8, torch.int8)}


def _dev(a, kind=np.int32):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a).astype(kind))).cuda()


def _stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


class Pool:
    """A pool [pages][kv][page][dim], optionally with room between heads and pages, a table and the view."""

    def __init__(self, qb, table, pages, kv, page, dim, store, room=0):
        import torch
        self.kind, self.dtype = _types(qb)[store]
        self.store, self.pages, self.kv, self.page, self.dim = store, pages, kv, page, dim
        self.table = np.asarray(table, np.int32)
        self.table_dev = _dev(self.table)
        heads = kv + (1 if room else 0)
        full = lambda *s: torch.full((*s, self.dtype.itemsize), DIRTY, dtype=torch.uint8, device="cuda").view(self.dtype)[..., 0]  # noqa: E731
        self.k_all, self.v_all = full(pages, heads, page + room, dim), full(pages, heads, page + room, dim)
        self.k, self.v = self.k_all[:, :kv, :page], self.v_all[:, :kv, :page]
        self.ks_all = self.vs_all = self.ks = self.vs = None
        if store in TOP:
            self.ks_all = torch.full((pages, heads, page + room), -7.0, device="cuda")
            self.vs_all = torch.full((pages, heads, page + room), -7.0, device="cuda")
            self.ks, self.vs = self.ks_all[:, :kv, :page], self.vs_all[:, :kv, :page]
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.view = qb.KVPages(p(self.k_all), p(self.v_all), p(self.ks_all), p(self.vs_all), self.table_dev.data_ptr(), self.k_all.stride(0),
                               self.k_all.stride(1), self.kind, pages, self.table.shape[0], kv, dim, page, self.table.shape[1])

    def fill(self, g, spread=1.0):
        import torch
        for x, s in ((self.k, self.ks), (self.v, self.vs)):
            r = torch.randn(x.shape, generator=g, device="cuda") * spread
            if s is None:
                x.copy_(r)
            else:
                a = r.abs().amax(-1)
                s.copy_(a / TOP[self.store])
                y = r / s[..., None]
                x.copy_(torch.round(y) if self.store == "int8" else y)
        return self

    def rows(self, seq, positions):
        """K and V of a sequence's positions in 64 bits, [kv][n][dim]; positions whose page is not there are left out."""
        import torch
        at = [p for p in positions if p // self.page < self.table.shape[1] and 0 <= self.table[seq, p // self.page] < self.pages]
        page = torch.tensor([int(self.table[seq, p // self.page]) for p in at], dtype=torch.long, device="cuda")
        row = torch.tensor([p % self.page for p in at], dtype=torch.long, device="cuda")
        out = []
        for x, s in ((self.k, self.ks), (self.v, self.vs)):
            y = x[page, :, row].float().double()
            out.append((y if s is None else y * s[page, :, row][..., None].double()).transpose(0, 1))
        return out

    def raw(self):
        import torch
        return [t.clone().view(torch.uint8) if t.dtype.itemsize == 1 else t.clone().view(torch.int16) if t.dtype.itemsize == 2
                else t.clone().view(torch.int32) for t in (self.k_all, self.v_all, self.ks_all, self.vs_all) if t is not None]


def _table(rng, needed, page, extra=0):
    """Tables of sequences that hold `needed` positions, pages in any order, and the pool's size."""
    count = [-(-n // page) for n in needed]
    table = np.full((len(needed), max(max(count), 1) + extra), -1, np.int32)
    pool = rng.permutation(sum(count) + 2)
    at = 0
    for r, n in enumerate(count):
        table[r, :n] = pool[at:at + n]
        at += n
    return table, len(pool)


# ---------------------------------------------------------------------------
# norms, rotation, rows to pages
# ---------------------------------------------------------------------------
def _rope64(x, gain, eps, base, positions):
    """Normalised and rotated rows [n][heads][dim] in 64 bits, and a bound on the fp32 form's error."""
    import torch
    d = x.shape[-1]
    y = x if gain is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain
    turn = positions.double()[:, None] * torch.tensor([base ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device="cuda")
    c, s = turn.cos()[:, None], turn.sin()[:, None]
    a, b = y[..., :d // 2], y[..., d // 2:]
    out = torch.cat([a * c - b * s, b * c + a * s], -1)
    # the mean's 16 + 3 sums, root, quotient and two products (24 roundings); the angle in half turns to 2^-25, so to pi 2^-25, sine
    # and cosine to 2 units, two products: 8 more, of |a| + |b|.  Angles here: pos * 2^-52 of the fp64 form's own
    tol = 40 * 2.0 ** -24 * (a.abs() + b.abs()) + (a.abs() + b.abs()) * positions.double()[:, None, None].abs() * 2.0 ** -51
    return out, torch.cat([tol, tol], -1)


def _codes64(x, store):
    """(codes as values, scale) of rows x in 64 bits: nearest code, ties to even, from the list of e4m3 values."""
    import torch
    a = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -60)
    y = x * TOP[store] / a
    if store == "int8":
        return torch.round(y), a / TOP[store]
    n = torch.arange(127, device=x.device)
    e, m = n >> 3, (n & 7).double()
    values = torch.where(e == 0, m / 512, (1 + m / 8) * torch.exp2(e - 7.0))
    z = y.abs()
    hi = torch.searchsorted(values, z.contiguous()).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    down, up = z - values[lo], values[hi] - z
    return torch.where((down < up) | ((down == up) & (lo % 2 == 0)), values[lo], values[hi]) * y.sign(), a / TOP[store]


def _rope(qb, pool, q, k, v, gains, gain_kind, eps, base, positions, seqs, out, with_k, pad=0, stream=None):
    """Runs the call; q, k, v [n][heads][dim].  Rows of inputs and outputs have `pad` elements behind them."""
    import torch
    n, heads, dim = q.shape
    kinds = {torch.bfloat16: qb.BF16, torch.float16: qb.FP16, torch.float32: qb.FP32}

    def padded(x):
        y = torch.full((n, x.shape[1] * dim + pad), float("nan"), dtype=x.dtype, device="cuda")
        y[:, :x.shape[1] * dim] = x.reshape(n, -1)
        return y

    qs, ks, vs = padded(q), padded(k), padded(v)
    qo = torch.full((n, heads * dim + pad), 7.0, dtype=out, device="cuda")
    ko = torch.full((n, k.shape[1] * dim + pad), 7.0, dtype=out, device="cuda")
    pos, sq = _dev(positions), _dev(seqs)
    g = [None, None] if gains is None else [x.contiguous() for x in gains]
    qb.qk_rope(qs.data_ptr(), ks.data_ptr(), vs.data_ptr() if pool else 0, kinds[q.dtype], qs.stride(0), ks.stride(0), vs.stride(0), n, heads, k.shape[1], dim,
               0 if gains is None else g[0].data_ptr(), 0 if gains is None else g[1].data_ptr(), gain_kind, eps, base, pos.data_ptr(), qo.data_ptr(),
               ko.data_ptr() if with_k else 0, kinds[out], qo.stride(0), ko.stride(0), pool.view if pool else None, sq.data_ptr() if pool else 0,
               _stream() if stream is None else stream)
    torch.cuda.synchronize()
    assert bool((qo[:, heads * dim:] == 7).all()) and bool((ko[:, k.shape[1] * dim:] == 7).all())
    return qo[:, :heads * dim].view(n, heads, dim), ko[:, :k.shape[1] * dim].view(n, k.shape[1], dim)


@pytest.mark.parametrize("src", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("store,out", [("bf16", "bf16"), ("fp16", "fp32"), ("e4m3", "fp16"), ("int8", "bf16")])
@pytest.mark.parametrize("n,heads,kv,dim,page,gain,pad", [(1, 16, 8, 128, 16, "bf16", 0), (131, 6, 3, 64, 8, "fp32", 8), (67, 5, 5, 128, 1, "fp16", 16),
                                                          (1029, 4, 1, 64, 64, None, 0), (4099, 2, 1, 128, 32, "bf16", 8)])
def test_rope_rows_and_pages(qb, src, store, out, n, heads, kv, dim, page, gain, pad):
    """Q and K rows, and K and V in their pages, against the definition; everything else of the pool stays as it was."""
    import torch
    g, rng = _gen(n), np.random.RandomState(n)
    kind, dtype = _types(qb)[src]
    kind_out, out_dtype = _types(qb)[out]
    b = 3
    seqs = np.sort(rng.randint(0, b, n))
    first = [5, 0, 17]
    positions = np.zeros(n, np.int64)
    for s in range(b):
        at = np.flatnonzero(seqs == s)
        positions[at] = first[s] + np.arange(len(at))
    table, pages = _table(rng, [n + 20] * b, page)
    pool = Pool(qb, table, pages, kv, page, dim, store, room=2)
    q, k, v = ((torch.randn(n, h, dim, generator=g, device="cuda") * 3).to(dtype) for h in (heads, kv, kv))
    gains = None if gain is None else [(1 + 0.5 * torch.randn(dim, generator=g, device="cuda")).to(_types(qb)[gain][1]) for _ in range(2)]
    before = [t.clone() for t in (pool.k_all, pool.v_all)]
    qo, ko = _rope(qb, pool, q, k, v, gains, 9 if gain is None else _types(qb)[gain][0], 1e-6, 1e6, positions, seqs, out_dtype, True, pad)
    pos = _dev(positions, np.int64)
    half = torch.finfo(out_dtype).eps / 2
    rows = {}
    for name, x, got in (("q", q, qo), ("k", k, ko)):
        want, tol = _rope64(x.double(), None if gains is None else gains[name == "k"].double(), 1e-6, 1e6, pos)
        rows[name] = want, tol
        err = (got.double() - want).abs()
        assert bool((err <= tol * (1 + half) + half * want.abs() + 2.0 ** -25).all()), float((err - half * want.abs()).max())
    page_no = torch.from_numpy(table[seqs, positions // page].astype(np.int64)).cuda()
    row = pos % page
    got_k, got_v = (pool.k[page_no, :, row].float().double(), pool.v[page_no, :, row].float().double())
    if store in TOP:
        want_v, a = _codes64(v.double(), store)
        assert torch.equal(got_v, want_v) and torch.equal(pool.vs[page_no, :, row], a[..., 0].float())
        scale = pool.ks[page_no, :, row][..., None].double()
        want, tol = rows["k"]
        amax = want.abs().amax(-1, keepdim=True)
        worst = tol.amax(-1, keepdim=True)
        assert bool(((scale * TOP[store] - amax).abs() <= worst + 2.0 ** -22 * amax).all())
        # half a step of the code, what the scale and the value are off by
        step = (want.abs() * 2.0 ** -4).clamp_min(2.0 ** -10 * amax / 448) if store == "e4m3" else amax / 127 / 2
        assert bool(((got_k * scale - want).abs() <= step * (1 + 2.0 ** -10) + 2 * worst + 2.0 ** -20 * amax).all())
    else:
        assert torch.equal(got_v, v.to(pool.dtype).double())
        want, tol = rows["k"]
        half = torch.finfo(pool.dtype).eps / 2
        assert bool(((got_k - want).abs() <= tol * (1 + half) + half * want.abs() + 2.0 ** -25).all())
    for all_, x, old in ((pool.k_all, pool.k, before[0]), (pool.v_all, pool.v, before[1])):
        x[page_no, :, row] = torch.zeros((), dtype=pool.dtype, device="cuda") if store not in TOP else x[page_no, :, row]
        y, z = all_.clone().view(torch.uint8), old.clone().view(torch.uint8)
        mask = torch.zeros(all_.shape, dtype=torch.bool, device="cuda")
        mask[:, :kv, :page][page_no, :, row] = True
        mask = mask[..., None].expand(*mask.shape, pool.dtype.itemsize).reshape(y.shape)
        assert torch.equal(y[~mask], z[~mask])
    if store in TOP:
        keep = torch.ones_like(pool.ks_all, dtype=torch.bool)
        keep[:, :kv, :page][page_no, :, row] = False
        assert bool((pool.ks_all[keep] == -7).all()) and bool((pool.vs_all[keep] == -7).all())


@pytest.mark.parametrize("base", [1e6, 10000.0, 1.0])
def test_rope_far_positions(qb, base):
    """Angles of positions up to 2^31 - 1, against whole-number arithmetic on the host."""
    from decimal import Decimal, getcontext
    import torch
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    positions = [0, 1, 32767, 1048575, 123456789, 2 ** 31 - 1]
    dim, n = 64, len(positions)
    x = torch.zeros(n, 1, dim, device="cuda")
    x[..., :dim // 2] = 1.0                                # so the halves become cosine and sine
    qo, _ = _rope(qb, None, x, x, x, None, 0, 0.0, base, positions, [0] * n, torch.float32, False)
    for r, p in enumerate(positions):
        for j in range(dim // 2):
            turns = Decimal(p) * (Decimal(base) ** (Decimal(-2 * j) / dim)) / (2 * pi)
            a = float((turns - turns.to_integral_value()) * 2 * pi)
            # a turn to 2^-64 * position, pi 2^-24 of the conversion, 2 units of sine and cosine
            tol = 6.3 * p * 2.0 ** -63 + 4 * 2.0 ** -24 + 2.0 ** -22
            assert abs(float(qo[r, 0, j]) - math.cos(a)) <= tol and abs(float(qo[r, 0, dim // 2 + j]) - math.sin(a)) <= tol, (p, j)


@pytest.mark.parametrize("store", ["bf16", "e4m3"])
def test_rope_left_out_rows(qb, store):
    """Negative positions are left out altogether; sequences, positions and pages that are not there reach no page."""
    import torch
    g = _gen(2)
    table = [[0, -1, 99], [2, 3, 4]]
    pool = Pool(qb, table, 5, 2, 8, 64, store)
    before = pool.raw()
    positions = [-1, 9, 17, 24, 3, 5, -2 ** 31, 2 ** 31 - 1, 1]
    seqs = [0, 0, 0, 1, 2, -1, 1, 1, -2 ** 31]
    x = [torch.randn(len(seqs), 2, 64, generator=g, device="cuda").bfloat16() for _ in range(3)]
    qo, ko = _rope(qb, pool, *x, None, 0, 1e-6, 1e4, positions, seqs, torch.bfloat16, True)
    for a, b in zip(before, pool.raw()):
        assert torch.equal(a, b)
    gone = torch.tensor([p < 0 for p in positions], device="cuda")
    assert bool((qo[gone] == 7).all()) and bool((ko[gone] == 7).all()) and not bool((qo[~gone] == 7).all(-1).any())


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_rope_rows_that_are_not_finite(qb, store):
    """An infinity or NaN spoils its own head's row alone; an 8-bit row that holds one reads back as NaN; zero rows stay zero."""
    import torch
    pool = Pool(qb, [[1, 0]], 2, 2, 4, 64, store)
    x = [torch.ones(4, 2, 64, device="cuda") for _ in range(3)]
    x[0][0, 0, 3], x[1][1, 1, 5], x[2][2, 0, 63], x[1][3] = float("nan"), float("inf"), float("-inf"), 0.0
    qo, ko = _rope(qb, pool, *x, [torch.ones(64, device="cuda")] * 2, qb.FP32, 1e-6, 1e4, [0, 1, 4, 7], [0] * 4, torch.float32, True)
    bad_q, bad_k = qo.isnan().any(-1), ko.isnan().any(-1)
    assert bad_q.sum() == 1 and bad_q[0, 0] and bad_k.sum() == 1 and bad_k[1, 1] and bool((ko[3] == 0).all())
    k, v = pool.rows(0, [0, 1, 4, 7])
    assert bool((~k.isfinite()).any(-1).nonzero().tolist() == [[1, 1]]) and bool((~v.isfinite()).any(-1).nonzero().tolist() == [[0, 2]])
    assert bool((k[:, 3] == 0).all())


# ---------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------
def _bounded(x, k, v, scale, seen, dtype, wide):
    """softmax(scale x k) v of [h][n][dim] rows over [h][m][dim] keys where seen [n][m], and a bound on a kernel's error: the
    weights' and the output's roundings to 16 bits (half a step each), fp32 scores, exp2's argument and result."""
    import torch
    half, dim = torch.finfo(dtype).eps / 2, x.shape[-1]
    half_p = torch.finfo(torch.float16).eps / 2 if wide else half
    s = x @ k.transpose(-1, -2) * scale
    w = torch.softmax(torch.where(seen, s, -math.inf), -1)
    w = torch.where(seen.any(-1)[:, None], w, 0.0)
    size = torch.where(seen, x.abs() @ k.abs().transpose(-1, -2) * abs(scale), 0.0).amax(-1, keepdim=True)
    rel = half_p + 2 * (dim + 8) * 2.0 ** -24 * size + 2.0 ** -20
    o, av = w @ v, w @ v.abs()
    # fp16 weights below 2^-24 of the unit are lost: of the largest, or of 2^-8 of it
    lost = 2.0 ** -23 * k.shape[-2] * v.abs().amax(-2, keepdim=True) if wide or dtype == torch.float16 else 0.0
    return o, (rel * av + lost) * (1 + half) + half * o.abs() + 2.0 ** -24 * (dtype == torch.float16)


def _prompt(qb, q, k, v, starts, k_starts, scale, pad=0, shift=0, behind=0, stream=None):
    """Runs the call on rows with `pad` elements behind them, out starting `shift` elements into its buffer; `behind` rows of out follow."""
    import torch
    n, heads, dim = q.shape
    kind = qb.BF16 if q.dtype == torch.bfloat16 else qb.FP16

    def padded(x):
        y = torch.full((x.shape[0], x.shape[1] * dim + pad), float("nan"), dtype=x.dtype, device="cuda")
        y[:, :x.shape[1] * dim] = x.reshape(x.shape[0], -1)
        return y

    qs, ks, vs = padded(q), padded(k), padded(v)
    ld = heads * dim + pad
    buffer = torch.full((shift + (n + behind) * ld,), 5.0, dtype=q.dtype, device="cuda")
    st, kst = _dev(starts), None if k_starts is None else _dev(k_starts)
    qb.prompt_attention(qs.data_ptr(), ks.data_ptr(), vs.data_ptr(), buffer.data_ptr() + 2 * shift, kind, ld, ks.stride(0), vs.stride(0), ld, st.data_ptr(),
                        0 if kst is None else kst.data_ptr(), len(starts) - 1, n, k.shape[0], heads, k.shape[1], dim, scale,
                        _stream() if stream is None else stream)
    torch.cuda.synchronize()
    out = buffer[shift:].view(n + behind, ld)
    assert bool((buffer[:shift] == 5).all()) and bool((out[n:] == 5).all()) and bool((out[:, heads * dim:] == 5).all())
    return out[:n, :heads * dim].reshape(n, heads, dim)


def _check_prompt(qb, q, k, v, starts, k_starts, scale, **kw):
    import torch
    got = _prompt(qb, q, k, v, starts, k_starts, scale, **kw)
    kst = starts if k_starts is None else k_starts
    group = q.shape[1] // k.shape[1]
    covered = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for s in range(len(starts) - 1):
        a, b, ka, kb = starts[s], starts[s + 1], kst[s], kst[s + 1]
        if b <= a:
            continue
        covered[a:b] = True
        n, m = b - a, kb - ka
        if m == 0:
            assert bool((got[a:b] == 0).all())
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n)
        for h in range(k.shape[1]):
            x = q[a:b, h * group:(h + 1) * group].double().transpose(0, 1)
            want, tol = _bounded(x, k[ka:kb, h].double()[None], v[ka:kb, h].double()[None], scale, seen, q.dtype, False)
            err = (got[a:b, h * group:(h + 1) * group].double().transpose(0, 1) - want).abs()
            bad = ~(err <= tol)
            assert not bool(bad.any()), (s, h, int(bad.sum()), float((err / tol.clamp_min(1e-30))[bad].max()), bad.nonzero()[:4].tolist())
    assert bool((got[~covered] == 5).all())
    return got


def _rows(seed, n, heads, m, kv, dim, dtype):
    import torch
    g = _gen(seed)
    return [torch.randn(*s, dim, generator=g, device="cuda").to(dtype) for s in ((n, heads), (m, kv), (m, kv))]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,contexts,heads,kv,dim", [
    ([1], [0], 2, 1, 128), ([100], [0], 4, 2, 128), ([128, 128], [0, 0], 4, 2, 64), ([129, 0, 127, 1, 300], [0] * 5, 4, 4, 128),
    ([257, 64, 65], [0, 200, 63], 9, 3, 64), ([5, 70, 40], [1000, 0, 128], 16, 2, 128), ([33, 2], [127, 126], 5, 1, 128),
    ([40, 17], [0, 90], 48, 1, 64), ([3, 4, 5], [0, 1, 0], 128, 1, 128), ([700, 513], [0, 31], 8, 4, 128), ([1500], [0], 2, 2, 64)])
def test_prompt_ragged(qb, dtype, lens, contexts, heads, kv, dim):
    """Lengths around the tiles' ends, contexts, one to 128 query heads for each K/V head, rows behind the last sequence."""
    import torch
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    k_starts = np.concatenate([[0], np.cumsum(np.add(lens, contexts))]).tolist()
    q, k, v = _rows(len(lens) + heads, starts[-1] + 3, heads, k_starts[-1] + 2, kv, dim, _types(qb)[dtype][1])
    _check_prompt(qb, q, k, v, starts, k_starts, dim ** -0.5)
    if not any(contexts):
        _check_prompt(qb, q, k, v, starts, None, dim ** -0.5)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 2.0])
@pytest.mark.parametrize("pad,shift", [(8, 8), (24, 0)])
def test_prompt_scales_and_strides(qb, scale, pad, shift):
    import torch
    q, k, v = _rows(4, 210, 6, 290, 3, 64, torch.bfloat16)
    _check_prompt(qb, q, k, v, [3, 150, 210], [10, 200, 290], scale, pad=pad, shift=shift, behind=2)


def test_prompt_fewer_keys_than_queries(qb):
    """The first queries see no key: zeros."""
    import torch
    q, k, v = _rows(5, 400, 4, 300, 2, 128, torch.bfloat16)
    got = _check_prompt(qb, q, k, v, [0, 140, 300, 400], [0, 1, 100, 100], 0.1)
    assert bool((got[:139] == 0).all()) and bool((got[139] != 0).any()) and bool((got[300:] == 0).all())


def test_prompt_many_sequences(qb):
    """More sequences than a warp holds at once, many of them empty."""
    import torch
    rng = np.random.RandomState(3)
    lens = np.where(rng.rand(700) < 0.4, 0, rng.randint(1, 40, 700))
    lens[333] = 900
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v = _rows(6, starts[-1], 2, starts[-1], 1, 64, torch.float16)
    _check_prompt(qb, q, k, v, starts, None, 0.125)


def test_prompt_more_items_than_multiprocessors(qb):
    """Every CTA takes several items, of different lengths."""
    import torch
    lens = [2000, 1, 1300, 700, 90, 2500]
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v = _rows(7, starts[-1], 16, starts[-1], 8, 128, torch.bfloat16)
    _check_prompt(qb, q, k, v, starts, None, 128 ** -0.5)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_short_items_behind_long_ones(qb, dim):
    """CTAs go from items of many key tiles to items of one, where K and V change places in the ring of parts; again and again."""
    import torch
    lens = [3000, 1500] + [50] * 500 + [130] * 40
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v = _rows(17, starts[-1], 8, starts[-1], 4, dim, torch.bfloat16)
    want = _check_prompt(qb, q, k, v, starts, None, dim ** -0.5)
    for _ in range(40):
        assert torch.equal(_prompt(qb, q, k, v, starts, None, dim ** -0.5), want)


def test_prompt_repeats_give_the_same_bits(qb):
    """Many calls one behind the other, with other inputs in between: no order of arrival shows."""
    import torch
    sets = [_rows(20 + i, 4096, 16, 4096, 8, 128, torch.bfloat16) for i in range(3)]
    st = _dev([0, 4096])
    call = lambda q, k, v, o: qb.prompt_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), qb.BF16, 2048, 1024, 1024, 2048, st.data_ptr(), 0, 1, 4096,  # noqa: E731
                                                  4096, 16, 8, 128, 0.09, _stream())
    want = []
    for s in sets:
        want.append(torch.empty_like(s[0]))
        call(*s, want[-1])
    outs = [torch.empty_like(s[0]) for s in sets]
    for _ in range(100):
        for s, o in zip(sets, outs):
            o.fill_(1)
            call(*s, o)
        for o, w in zip(outs, want):
            assert torch.equal(o, w) and bool(w.isfinite().all())


@pytest.mark.parametrize("starts,k_starts", [([0, 500, 90], [0, 500, 90]), ([-5, 60, 10 ** 9], [-(10 ** 9), 70, 2 ** 31 - 1]), ([90, 20, 30], [0, 0, 50])])
def test_prompt_starts_of_any_value(qb, starts, k_starts):
    """Starts outside the rows count as their ends, a start behind its end as no rows: nothing else is written."""
    import torch
    q, k, v = _rows(8, 120, 2, 130, 1, 64, torch.bfloat16)
    got = _prompt(qb, q, k, v, starts, k_starts, 0.1, behind=1)
    cut = lambda x, top: min(max(x, 0), top)  # noqa: E731
    for s in range(2):
        a, b, ka, kb = cut(starts[s], 120), cut(starts[s + 1], 120), cut(k_starts[s], 130), cut(k_starts[s + 1], 130)
        if b > a:
            alone = _prompt(qb, q[a:b].contiguous(), k[ka:max(kb, ka + 1)].contiguous(), v[ka:max(kb, ka + 1)].contiguous(), [0, b - a], [0, max(kb - ka, 0)], 0.1)
            assert torch.equal(got[a:b], alone)


def test_prompt_starts_that_overlap(qb):
    """Hundreds of sequences over the same rows, many times the work that starts in order can name: the call ends, writes nothing
    outside its rows, and the next one is right."""
    import torch
    n = 5000
    q, k, v = _rows(15, n, 2, n, 1, 64, torch.bfloat16)
    got = _prompt(qb, q, k, v, [0, n] * 300, None, 0.1, pad=8, behind=3)
    assert bool((got.isfinite()).all())
    _check_prompt(qb, q, k, v, [0, n], None, 0.1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("what", ["nan", "inf", "lowest"])
def test_prompt_unseen_values_do_not_matter(qb, dtype, what):
    """Rows that a query does not see may hold anything: later ones of its own sequence, other sequences', those behind the last."""
    import torch
    dtype = _types(qb)[dtype][1]
    value = {"nan": float("nan"), "inf": float("inf"), "lowest": torch.finfo(dtype).min}[what]
    starts = [0, 70, 333]
    q, k, v = _rows(9, 340, 4, 340, 2, 128, dtype)
    plain = _prompt(qb, q, k, v, starts, None, 0.09)
    for at in (69, 70, 200, 255, 332, 335):
        k2, v2 = k.clone(), v.clone()
        k2[at:at + 1], v2[at:at + 1] = value, value
        if what != "lowest":
            v2[at, 1, 5] = -value
        got = _prompt(qb, q, k2, v2, starts, None, 0.09)
        end = 70 if at < 70 else 333 if at < 333 else at
        blind = torch.ones(340, dtype=torch.bool, device="cuda")
        blind[at:end] = False
        assert torch.equal(got[blind], plain[blind]), at
        if what == "nan":
            assert bool(got[at:end].isnan().all())


def test_prompt_infinite_values_that_are_seen(qb):
    """An infinity in V is the result of the rows that see it, in its column alone, also in the tile where some do not."""
    import torch
    q, k, v = _rows(10, 300, 2, 300, 1, 64, torch.bfloat16)
    want = _prompt(qb, q, k, v, [0, 300], None, 0.1)
    v[130, 0, 7], v[290, 0, 9], v[250, 0, 9] = float("inf"), float("inf"), float("-inf")
    got = _prompt(qb, q, k, v, [0, 300], None, 0.1)
    assert bool((got[130:, :, 7] == float("inf")).all()) and bool((got[250:290, :, 9] == float("-inf")).all()) and bool(got[290:, :, 9].isnan().all())
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[130:, :, 7] = keep[250:, :, 9] = False
    assert torch.equal(got[keep], want[keep])


def test_prompt_large_scores(qb):
    """Scores far apart and rising along the keys, so every tile raises the maximum; one key alone has all the weight."""
    import torch
    q, k, v = _rows(11, 700, 2, 700, 1, 128, torch.bfloat16)
    k = (k.float() * torch.linspace(0.1, 30, 700, device="cuda")[:, None, None]).bfloat16()
    _check_prompt(qb, q, k, v, [0, 700], None, 0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 4), (128, 4, 4), (64, 4, 2), (128, 8, 4)])
def test_prompt_maximum_that_rises_in_every_tile(qb, dtype, dim, heads, kv):
    """Keys that grow along each sequence, so that O is scaled in most tiles, beside the products of the tile's first half; several
    items a CTA, again and again: within the bounds, and always the same bits."""
    import torch
    lens = [2600, 1900, 900, 300] + [600] * 40
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v = _rows(31 + dim + heads, starts[-1], heads, starts[-1], kv, dim, _types(qb)[dtype][1])
    grow = torch.cat([torch.linspace(0.2, 24 * n / 1000 + 4, n) for n in lens]).cuda()
    k = (k.float() * grow[:, None, None]).to(k.dtype)
    want = _check_prompt(qb, q, k, v, starts, None, 0.4)
    for _ in range(30):
        assert torch.equal(_prompt(qb, q, k, v, starts, None, 0.4), want)


def test_prompt_long_items_are_not_waits_that_run_out(qb):
    """One query over two million keys: the warps of the second row tile have nothing to do for many times the limit of a wait, while
    the block makes progress all along."""
    import torch
    q, k, v = _rows(13, 1, 1, 1 << 21, 1, 64, torch.bfloat16)
    want = _prompt(qb, q, k, v, [0, 1], [0, 1 << 21], 0.125)
    assert bool(want.isfinite().all()) and bool((want != 0).any())
    qb.debug_draft_wait(1_000_000, -1)
    try:
        got = _prompt(qb, q, k, v, [0, 1], [0, 1 << 21], 0.125)
    finally:
        qb.debug_draft_wait()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_that_are_all_minus_infinity(qb, dtype):
    """A query whose scores are all -inf gets zeros, from prompts and from pages; one with a single score above -inf gets that key's values."""
    import torch
    dtype = _types(qb)[dtype][1]
    q, k, v = _rows(16, 200, 2, 200, 1, 64, dtype)
    q[..., 1], k[..., 1] = 1, -math.inf
    k[150, 0, 1] = 2
    got = _prompt(qb, q, k, v, [0, 200], None, 0.1)
    assert bool((got[:150] == 0).all()) and torch.equal(got[150:], v[150:151].expand(50, 2, 64))
    pool = Pool(qb, [[0, 1], [0, 1]], 2, 1, 128, 64, "bf16" if dtype == torch.bfloat16 else "fp16").fill(_gen(1))
    pool.k[0, 0], pool.k[1, 0, :72] = k[:128, 0], k[128:, 0]
    got = _attend(qb, pool, q[:2].contiguous(), [140, 190], 0.1)
    assert bool((got[0] == 0).all()) and torch.equal(got[1], pool.v[1, 0, 22].expand(2, 64))


@pytest.mark.parametrize("scale", [0.0, 2e-38, -2e-38])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_at_the_low_end(qb, scale, dim):
    """Products of queries and keys up to 10^38, which a scale near the smallest fp32 number, or of 0, brings back."""
    import torch
    q, k, v = _rows(18, 260, 4, 260, 2, dim, torch.bfloat16)
    _check_prompt(qb, q * 1e18, k * 1e18, v, [0, 260], None, scale)
    pool = Pool(qb, [list(range(20))] * 3, 20, 2, 16, dim, "bf16").fill(_gen(2))
    pool.k *= 1e18
    _check_paged(qb, pool, q[:3] * 1e18, [300, 40, 0], scale)


# One key with the weight 1, 8,191 with 2^-tail each and large values: the weights enter the product in fp16, whose steps
# below 2^-14 are 2^-24, in a unit of at most 2^-7 of the largest weight (8-bit pages: divided by the value's scale, at least a half of the
# unit's); half a step off each, beside the relative roundings: weight and result 2^-11 each, 2^-18 for exponents and sums.
def _far_tail(tail, eight_bits):
    keys, value = 8192, 512.0
    total = 1 + (keys - 1) * 2.0 ** -tail
    want = (keys - 1) * 2.0 ** -tail * value / total
    return keys, value, want, want * (2.0 ** -10 + 2.0 ** -18) + 2.0 ** -32 * keys * value * (2 if eight_bits else 1) + 2.0 ** -25


@pytest.mark.parametrize("tail", [12.0, 20.0, 24.5, 25.0, 28.0])
@pytest.mark.parametrize("first", [0, 100, 8191])
def test_prompt_many_small_weights_in_fp16(qb, tail, first):
    import torch
    keys, value, want, tol = _far_tail(tail, False)
    q = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda")
    k, v = torch.zeros(keys, 1, 64, dtype=torch.float16, device="cuda"), torch.full((keys, 1, 64), value, dtype=torch.float16, device="cuda")
    q[..., 3], k[..., 3], k[first], v[first] = 1, -tail, 0, 0
    got = _prompt(qb, q, k, v, [0, 1], [0, keys], math.log(2))
    assert bool(((got.double() - want).abs() <= tol).all()), (float(got[0, 0, 0]), want)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_reports_a_wait_that_ran_out(qb, dim):
    """K and V that are never announced: the bounded waits end, the call's rows are NaN, and the next call is right."""
    import torch
    q, k, v = _rows(12, 300, 4, 300, 2, dim, torch.bfloat16)
    qb.debug_draft_wait(5_000_000, 1)
    try:
        got = _prompt(qb, q, k, v, [0, 300], None, 0.1)
    finally:
        qb.debug_draft_wait()
    assert bool(got.isnan().all())
    _check_prompt(qb, q, k, v, [0, 300], None, 0.1)


@pytest.mark.parametrize("part,item", [(0, 1), (3, 2), (6, 4)])
def test_prompt_wait_that_ran_out_in_a_later_item(qb, part, item):
    """One-tile prompts, a few blocks more than others with the item whose part is never announced: every row of those blocks is NaN, those
    of the items before it too, and every other row is right."""
    import torch
    blocks = torch.cuda.get_device_properties(0).multi_processor_count
    n = (item - 1) * blocks + 40
    q, k, v = _rows(14, 5 * n, 2, 5 * n, 1, 64, torch.bfloat16)
    starts = list(range(0, 5 * n + 1, 5))
    want = _prompt(qb, q, k, v, starts, None, 0.1)
    qb.debug_draft_wait(5_000_000, part)
    try:
        got = _prompt(qb, q, k, v, starts, None, 0.1)
    finally:
        qb.debug_draft_wait()
    gone = got.isnan()
    assert torch.equal(torch.where(gone, 0, got), torch.where(gone, 0, want))
    rows = gone.view(n, -1)
    assert bool((rows.all(1) | ~rows.any(1)).all()) and int(rows.any(1).sum()) == 40 * item
    assert torch.equal(_prompt(qb, q, k, v, starts, None, 0.1), want)


# ---------------------------------------------------------------------------
# attention over pages
# ---------------------------------------------------------------------------
def _attend(qb, pool, q, lens, scale, pad=0, stream=None):
    import torch
    b, heads, dim = q.shape
    kind = qb.BF16 if q.dtype == torch.bfloat16 else qb.FP16
    qs = torch.full((b, heads * dim + pad), float("nan"), dtype=q.dtype, device="cuda")
    qs[:, :heads * dim] = q.reshape(b, -1)
    out = torch.full((b, heads * dim + pad), 5.0, dtype=q.dtype, device="cuda")
    work = torch.full((qb.paged_attention_workspace(pool.view, heads),), 0xFF, dtype=torch.uint8, device="cuda")   # NaN
    ln = _dev(lens)
    qb.paged_attention(pool.view, qs.data_ptr(), out.data_ptr(), kind, qs.stride(0), out.stride(0), heads, ln.data_ptr(), scale, work.data_ptr(),
                       work.numel(), _stream() if stream is None else stream)
    torch.cuda.synchronize()
    assert bool((out[:, heads * dim:] == 5).all())
    return out[:, :heads * dim].reshape(b, heads, dim)


def _check_paged(qb, pool, q, lens, scale, **kw):
    import torch
    got = _attend(qb, pool, q, lens, scale, **kw)
    b, heads, dim = q.shape
    capacity = pool.page * pool.table.shape[1]
    for r in range(b):
        k, v = pool.rows(r, range(int(lens[r]) + 1) if 0 <= lens[r] < capacity else [])
        if k.shape[1] == 0:
            assert bool((got[r] == 0).all())
            continue
        x = q[r].double().view(pool.kv, -1, dim)
        seen = torch.ones(x.shape[1], k.shape[1], dtype=torch.bool, device="cuda")
        want, tol = _bounded(x, k, v, scale, seen, q.dtype, pool.store in TOP)
        err = (got[r].double().view(want.shape) - want).abs()
        bad = ~(err <= tol)
        assert not bool(bad.any()), (r, int(lens[r]), int(bad.sum()), float((err / tol.clamp_min(1e-30))[bad].max()), bad.nonzero()[:4].tolist())
    return got


@pytest.mark.parametrize("store", ["16", "e4m3", "int8"])
@pytest.mark.parametrize("qt", ["bf16", "fp16"])
@pytest.mark.parametrize("kv,group,dim,page", [(2, 1, 128, 16), (1, 2, 64, 1), (3, 7, 64, 8), (2, 8, 128, 128), (1, 9, 128, 4), (2, 16, 64, 32), (1, 40, 128, 64)])
def test_paged_ragged_batches(qb, store, qt, kv, group, dim, page):
    """Lengths from none to several tiles, ends inside pages and tiles, sequences that are idle."""
    import torch
    rng, g = np.random.RandomState(group), _gen(group)
    lens = [0, 1, 15, 16, 63, 64, 127, 300, 517, -1, -2 ** 31, 2 ** 31 - 1]
    table, pages = _table(rng, [max(0, n + 1) if n < 1000 else 30 for n in lens], page, extra=1)
    pool = Pool(qb, table, pages, kv, page, dim, qt if store == "16" else store, room=1).fill(g)
    q = torch.randn(len(lens), kv * group, dim, generator=g, device="cuda").to(_types(qb)[qt][1])
    _check_paged(qb, pool, q, lens, dim ** -0.5, pad=8)


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("b,kv,group,dim,page,longest", [(1, 8, 2, 128, 16, 1024), (1, 1, 1, 64, 64, 9000), (5, 2, 3, 128, 32, 4100), (150, 2, 4, 64, 16, 900),
                                                         (3, 1, 20, 128, 256, 3000), (40, 8, 2, 128, 64, 700)])
def test_paged_shared_out(qb, store, b, kv, group, dim, page, longest):
    """Lines of tiles shared out over all SMs: single long sequences, ragged batches, several blocks of rows."""
    import torch
    rng, g = np.random.RandomState(b), _gen(b)
    lens = rng.randint(-1, longest, b)
    lens[0] = longest
    table, pages = _table(rng, lens + 1, page)
    pool = Pool(qb, table, pages, kv, page, dim, store).fill(g)
    q = torch.randn(b, kv * group, dim, generator=g, device="cuda").bfloat16()
    _check_paged(qb, pool, q, lens, dim ** -0.5)


@pytest.mark.parametrize("store", ["fp16", "e4m3", "int8"])
def test_paged_pages_that_are_not_there(qb, store):
    """Positions of missing pages have no part, wherever they lie; pages may serve several sequences; any order."""
    import torch
    g = _gen(4)
    table = np.array([[3, -1, 7, 1, 99, 2], [3, 3, 3, 5, 5, 6], [-1, -5, 2 ** 31 - 1, -1, -1, -1], [8, 4, 8, 0, -1, -1]], np.int32)
    for page in (2, 16, 32, 128):
        pool = Pool(qb, table, 9, 2, page, 128, store).fill(g)
        q = torch.randn(4, 6, 128, generator=g, device="cuda").to(torch.float16)
        for lens in ([6 * page - 1] * 4, [page, page - 1, 3 * page, 4 * page + 1], [0, 2 * page + 1, 6 * page, 4 * page]):
            _check_paged(qb, pool, q, lens, 0.1)


@pytest.mark.parametrize("store", ["bf16", "fp16", "e4m3", "int8"])
@pytest.mark.parametrize("length", [3, 40, 700])
def test_paged_unseen_values_do_not_matter(qb, store, length):
    """What lies behind a sequence's length in its pages, and in the pool's other pages, may be anything, scales included."""
    import torch
    g, rng = _gen(length), np.random.RandomState(1)
    table, pages = _table(rng, [length + 33] * 2, 16)
    pool = Pool(qb, table, pages, 2, 16, 128, store).fill(g)
    q = torch.randn(2, 4, 128, generator=g, device="cuda").to(torch.float16 if store == "fp16" else torch.bfloat16)
    lens = [length, length // 2]
    want = _attend(qb, pool, q, lens, 0.1)
    seen = torch.zeros(pages, 16, dtype=torch.bool, device="cuda")
    for r in range(2):
        for p in range(lens[r] + 1):
            seen[table[r, p // 16], p % 16] = True
    hidden = ~seen[:, None].expand(pages, 2, 16)
    for x, s in ((pool.k, pool.ks), (pool.v, pool.vs)):
        if store == "int8":
            x[hidden] = -128
        else:
            x[hidden] = torch.full((128,), float("nan"), device="cuda").to(x.dtype)
        if s is not None:
            s[hidden] = float("nan")
    assert torch.equal(_attend(qb, pool, q, lens, 0.1), want)


def test_paged_infinity_that_is_seen(qb):
    import torch
    g = _gen(6)
    pool = Pool(qb, [[0, 1, 2, 3]], 4, 1, 32, 64, "bf16").fill(g)
    pool.v[2, 0, 5, 9] = float("inf")
    q = torch.randn(1, 2, 64, generator=g, device="cuda").bfloat16()
    got = _attend(qb, pool, q, [100], 0.1)
    assert bool((got[..., 9] == float("inf")).all()) and bool(got[..., :9].isfinite().all()) and bool(got[..., 10:].isfinite().all())
    assert bool(_attend(qb, pool, q, [68], 0.1).isfinite().all())
    pool.k[0, 0, 0, 0] = float("nan")
    assert bool(_attend(qb, pool, q, [100], 0.1).isnan().all())


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("low,high", [(-40, -20), (-30, 10), (5, 30)])
def test_paged_value_scales_of_any_size(qb, store, low, high):
    """Value scales that differ by many powers of two, the largest anywhere; errors count against the largest value in sight."""
    import torch
    g, rng = _gen(8), np.random.RandomState(2)
    table, pages = _table(rng, [900, 40], 16)
    pool = Pool(qb, table, pages, 2, 16, 128, store).fill(g)
    pool.vs *= torch.exp2(torch.randint(low, high, pool.vs.shape, generator=g, device="cuda").float())
    q = torch.randn(2, 4, 128, generator=g, device="cuda").bfloat16()
    _check_paged(qb, pool, q, [899, 39], 0.1)


@pytest.mark.parametrize("store", ["bf16", "e4m3"])
def test_paged_large_scores(qb, store):
    """Scores that rise along the keys, so that the running base follows again and again; and queries of any magnitude."""
    import torch
    g = _gen(9)
    pool = Pool(qb, [list(range(40))], 40, 1, 32, 128, store).fill(g)
    if store == "bf16":
        pool.k.copy_(pool.k.float() * torch.linspace(0.1, 30, 1280, device="cuda").view(40, 1, 32, 1))
    else:
        pool.ks *= torch.linspace(0.1, 30, 1280, device="cuda").view(40, 1, 32)
    for size in (1.0, 2.0 ** -100, 2.0 ** 60):
        q = (torch.randn(1, 4, 128, generator=g, device="cuda") * size).bfloat16()
        _check_paged(qb, pool, q, [1270], 0.5 / size)
        _check_paged(qb, pool, q, [1270], -0.5 / size)


@pytest.mark.parametrize("tail", [12.0, 20.0, 24.5, 25.0, 28.0])
@pytest.mark.parametrize("store", ["fp16", "e4m3", "int8"])
@pytest.mark.parametrize("copies", [1, 40])
def test_paged_many_small_weights_in_fp16(qb, store, tail, copies):
    """Alone (a cluster, or shares of the line, an item) and 40 at once."""
    import torch
    keys, value, want, tol = _far_tail(tail, store != "fp16")
    pool = Pool(qb, np.tile(np.arange(keys // 64), (copies, 1)), keys // 64, 1, 64, 64, store)
    one = 1.0 if store == "fp16" else TOP[store]            # 8 bits: code times scale
    pool.k.copy_(torch.zeros(pool.k.shape, device="cuda"))
    pool.v.copy_(torch.full(pool.v.shape, value if store == "fp16" else one, device="cuda"))
    pool.k[..., 3] = torch.tensor(-tail if store == "fp16" else -one, device="cuda").to(pool.dtype)
    pool.k[1, 0, 36], pool.v[1, 0, 36] = (torch.zeros(64, device="cuda").to(pool.dtype) for _ in range(2))
    if store != "fp16":
        pool.ks.fill_(tail / one)
        pool.vs.fill_(value / one)
    q = torch.zeros(copies, 2, 64, dtype=torch.float16, device="cuda")
    q[..., 3] = 1
    got = _attend(qb, pool, q, [keys - 1] * copies, math.log(2))
    assert bool(((got.double() - want).abs() <= tol).all()), (float(got[0, 0, 0]), want)


def test_paged_beyond_32_bit_offsets(qb):
    """A pool whose pages lie more than 2^32 elements apart."""
    import torch
    g = _gen(10)
    dim, page, n = 64, 16, 5
    stride = (1 << 31) // n // dim * dim + 64 * dim
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs a large GPU")
    k, v = (torch.empty(n * stride * 2, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = _dev([[4, 0, 3]])
    pool = Pool(qb, [[4, 0, 3]], n, 1, page, dim, "bf16").fill(g)
    for p in range(n):
        k[2 * p * stride:2 * p * stride + page * dim] = pool.k[p].reshape(-1)
        v[2 * p * stride:2 * p * stride + page * dim] = pool.v[p].reshape(-1)
    assert 2 * 4 * stride > 1 << 31
    q = torch.randn(1, 2, dim, generator=g, device="cuda").bfloat16()
    want = _attend(qb, pool, q, [45], 0.1)
    pool.view = qb.KVPages(k.data_ptr(), v.data_ptr(), None, None, table.data_ptr(), 2 * stride, page * dim, qb.BF16, n, 1, 1, dim, page, 3)
    assert torch.equal(_attend(qb, pool, q, [45], 0.1), want)


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def _score(qb, logits, tokens, temp, top, entropy=True, stream=None):
    import torch
    n, vocab = logits.shape
    kind = {torch.bfloat16: qb.BF16, torch.float16: qb.FP16, torch.float32: qb.FP32}[logits.dtype]
    lp, en = torch.full((n,), 9.0, device="cuda"), torch.full((n,), 9.0, device="cuda")
    ids, tl = torch.full((n, top), -9, dtype=torch.int32, device="cuda"), torch.full((n, top), 9.0, device="cuda")
    tk = None if tokens is None else _dev(tokens)
    qb.token_logprobs(logits.data_ptr(), kind, logits.stride(0), n, vocab, 0 if tk is None else tk.data_ptr(), temp, top, 0 if tk is None else lp.data_ptr(),
                      en.data_ptr() if entropy else 0, ids.data_ptr() if top else 0, tl.data_ptr() if top else 0, _stream() if stream is None else stream)
    torch.cuda.synchronize()
    return lp, en, ids, tl


def _check_score(qb, logits, tokens, temp, top):
    """Against 64 bits: ids exactly; sums of up to vocab / 512 + 600 fp32 terms a thread and block, scores to two roundings each."""
    import torch
    lp, en, ids, tl = _score(qb, logits, tokens, temp, top)
    n, vocab = logits.shape
    unit = 2.0 ** -24
    sums = (vocab / 512 + 700) * unit
    for r in range(n):
        x = logits[r].double()
        y = torch.log_softmax(x / temp, 0)
        h = -torch.special.xlogy(y.exp(), y.exp()).sum()
        if tokens is not None:
            t = int(tokens[r])
            if 0 <= t < vocab:
                want = float(y[t])
                assert float(lp[r]) == want or abs(float(lp[r]) - want) <= sums + 4 * unit * (abs(want) + 20), (r, float(lp[r]), want)
            else:
                assert math.isnan(float(lp[r]))
        # the mean of y: relative to the entropy and the sums' error
        assert abs(float(en[r]) - float(h)) <= 2 * sums * (1 + float(h)) + 16 * unit * float(h), (r, float(en[r]), float(h))
        order = torch.sort(logits[r].float() + 0.0, descending=True, stable=True).indices[:top]
        k = len(order)
        assert ids[r, :k].tolist() == order.tolist(), r
        assert bool((ids[r, k:] == -1).all()) and bool((tl[r, k:] == -math.inf).all())
        want = y[order]
        same = tl[r, :k].double() == want
        assert bool((same | ((tl[r, :k].double() - want).abs() <= sums + 4 * unit * (want.abs() + 20))).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,vocab,pad,shift,top", [(1, 151936, 0, 0, 20), (3, 151937, 3, 1, 64), (40, 5003, 0, 0, 5), (200, 32000, 16, 0, 1), (2, 1, 0, 0, 3), (5, 7, 0, 1, 10),
                                                   (9, 1000, 1, 3, 0), (1, 262147, 0, 1, 33), (310, 4096, 0, 0, 64)])
def test_logprobs(qb, dtype, n, vocab, pad, shift, top):
    """Sizes of all alignments, one row to hundreds, tokens outside the vocabulary."""
    import torch
    g, rng = _gen(vocab), np.random.RandomState(n)
    dtype = _types(qb)[dtype][1]
    buffer = torch.full((shift + n * (vocab + pad),), float("nan"), device="cuda", dtype=dtype)
    logits = buffer[shift:].view(n, vocab + pad)[:, :vocab]
    logits.copy_(torch.randn(n, vocab, generator=g, device="cuda") * 4)
    tokens = rng.randint(0, vocab, n)
    tokens[-1] = -1 if n % 2 else vocab
    _check_score(qb, logits, tokens, 0.7, top)


@pytest.mark.parametrize("temp", [1e-6, 0.05, 1.0, 30.0, 1e6])
def test_logprobs_temperatures(qb, temp):
    import torch
    logits = torch.randn(4, 20011, generator=_gen(1), device="cuda") * (0.001 if temp < 0.01 else 4)
    lp, en, ids, tl = _score(qb, logits, [1, 2, 3, 20010], temp, 4)
    for r, t in enumerate([1, 2, 3, 20010]):
        y = torch.log_softmax(logits[r].double() / temp, 0)
        # the factor log2(e) / temperature is one fp32 number: 2^-24 of a score
        assert abs(float(lp[r]) - float(y[t])) <= (20011 / 512 + 700) * 2.0 ** -24 + 2.0 ** -22 * (abs(float(y[t])) + 20)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [1, 5, 300])
def test_logprobs_masked_and_equal_logits(qb, dtype, n):
    """Rows of which a few logits are above -inf, or the type's lowest value, all equal, ascending, or of few values: ids by value, then index."""
    import torch
    dtype = _types(qb)[dtype][1]
    g, vocab = _gen(n), 40009
    for kind in ("few", "lowest", "equal", "zeros", "ascending", "descending", "steps", "one"):
        x = torch.randn(n, vocab, generator=g, device="cuda")
        if kind in ("few", "lowest"):
            keep = torch.rand(n, vocab, generator=g, device="cuda") < 20 / vocab
            keep[:, 17] = True
            x = torch.where(keep, x, -math.inf if kind == "few" else torch.finfo(dtype).min)
        elif kind == "equal":
            x[:] = torch.finfo(dtype).min
        elif kind == "zeros":
            x = torch.where(x > 0, 0.0, -0.0)
        elif kind in ("ascending", "descending"):
            x[:] = torch.linspace(-3, 3, vocab, device="cuda") * (1 if kind == "ascending" else -1)
        elif kind == "steps":
            x = torch.round(x)
        else:
            x[:] = -math.inf
            x[:, vocab - 2] = 3.0
        x = x.to(dtype)
        for top in (1, 7, 64):
            _check_score(qb, x if n < 10 else x[:10].contiguous(), np.full(min(n, 10), 17), 1.0, top)
        if n > 10:                                          # (as many rows as make one block a row)
            a, b = _score(qb, x, None, 1.0, 20), _score(qb, x[:5].contiguous(), None, 1.0, 20)
            assert torch.equal(a[2][:5], b[2])


@pytest.mark.parametrize("n", [1, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -math.inf])
def test_logprobs_rows_without_a_distribution(qb, n, bad):
    import torch
    x = torch.randn(n, 30011, generator=_gen(2), device="cuda")
    clean = _score(qb, x, [3] * n, 1.0, 5)
    at = n // 2
    if bad == -math.inf:
        x[at] = bad
    else:
        x[at, 29999] = bad
    lp, en, ids, tl = _score(qb, x, [3] * n, 1.0, 5)
    assert math.isnan(float(lp[at])) and math.isnan(float(en[at])) and ids[at].tolist() == [-1] * 5 and bool(tl[at].isnan().all())
    keep = torch.arange(n, device="cuda") != at
    for a, b in zip(clean, (lp, en, ids, tl)):
        assert torch.equal(a[keep], b[keep])


def test_logprobs_of_an_engine(qb, engine):
    """The step's own logits on the device, scored on the engine's stream."""
    import torch
    logits = engine.forward(11, 0)
    lp, en, ids = torch.empty(1, device="cuda"), torch.empty(1, device="cuda"), torch.empty(1, 3, dtype=torch.int32, device="cuda")
    tl = torch.empty(1, 3, device="cuda")
    tk = _dev([42])
    torch.cuda.synchronize()
    qb.token_logprobs(engine.device_logits_ptr(), qb.FP32, qb.VOCAB_SIZE, 1, qb.VOCAB_SIZE, tk.data_ptr(), 1.0, 3, lp.data_ptr(), en.data_ptr(), ids.data_ptr(),
                      tl.data_ptr(), engine.stream)
    torch.cuda.synchronize()
    y = torch.log_softmax(torch.from_numpy(logits).double(), 0)
    assert abs(float(lp[0]) - float(y[42])) <= 1e-4 and ids[0].tolist() == torch.sort(y, descending=True, stable=True).indices[:3].tolist()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
class Layer:
    """Projections of one attention layer as numbers: what a server would have from its matrix products."""

    def __init__(self, heads, kv, dim, n, seed, dtype):
        import torch
        g = _gen(seed)
        self.heads, self.kv, self.dim = heads, kv, dim
        self.q, self.k, self.v = (torch.randn(n, h * dim, generator=g, device="cuda").to(dtype) for h in (heads, kv, kv))
        self.gains = [(1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).bfloat16() for _ in range(2)]

    def rope(self, qb, rows, positions, seqs, pool, stream=None):
        """Rows of the packed order through qk_rope: q and k as 16-bit rows, k and v in the pages."""
        import torch
        n, kind = len(rows), qb.BF16 if self.q.dtype == torch.bfloat16 else qb.FP16
        q, k, v = (x[rows].contiguous() for x in (self.q, self.k, self.v))
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        pos, sq = _dev(positions), _dev(seqs)
        qb.qk_rope(q.data_ptr(), k.data_ptr(), v.data_ptr(), kind, self.heads * self.dim, self.kv * self.dim, self.kv * self.dim, n, self.heads, self.kv, self.dim,
                   self.gains[0].data_ptr(), self.gains[1].data_ptr(), qb.BF16, 1e-6, 1e6, pos.data_ptr(), qo.data_ptr(), ko.data_ptr(), kind, self.heads * self.dim,
                   self.kv * self.dim, pool.view, sq.data_ptr(), _stream() if stream is None else stream)
        torch.cuda.synchronize()
        return qo.view(n, self.heads, self.dim), ko.view(n, self.kv, self.dim), v.view(n, self.kv, self.dim)


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_prompt_then_steps(qb, store):
    """Prompts enter the pages and attend to themselves; then a token a step for every sequence.  Over 16-bit pages each step's
    rows are those of the prompt attention over the whole sequence, within both calls' bounds; over 8-bit pages the
    definition's over the quantised rows.  The rows' scores feed the log probabilities, whose best token is the one that
    greedy verification takes."""
    import torch
    lens, steps, heads, kv, dim, page = [70, 1, 200], 5, 4, 2, 128, 16
    total = [n + steps for n in lens]
    first = np.concatenate([[0], np.cumsum(total)])
    layer = Layer(heads, kv, dim, int(first[-1]), 3, torch.bfloat16)
    table, pages = _table(np.random.RandomState(0), total, page)
    pool = Pool(qb, table, pages, kv, page, dim, store)
    rows = np.concatenate([first[s] + np.arange(n) for s, n in enumerate(lens)])
    q, k, v = layer.rope(qb, rows, np.concatenate([np.arange(n) for n in lens]), np.repeat(np.arange(3), lens), pool)
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    _check_prompt(qb, q, k, v, starts, None, dim ** -0.5)
    whole = Pool(qb, table, pages, kv, page, dim, "bf16")
    every = layer.rope(qb, np.arange(first[-1]), np.concatenate([np.arange(n) for n in total]), np.repeat(np.arange(3), total), whole)
    reference = _check_prompt(qb, *every, first.tolist(), None, dim ** -0.5)
    head = torch.randn(heads * dim, 5000, generator=_gen(5), device="cuda")
    for i in range(steps):
        at = [n + i for n in lens]
        q, _, _ = layer.rope(qb, first[:3] + at, at, np.arange(3), pool)
        got = _check_paged(qb, pool, q, at, dim ** -0.5)
        if store == "bf16":
            k64, v64 = pool.rows(2, range(at[2] + 1))
            seen = torch.ones(heads // kv, at[2] + 1, dtype=torch.bool, device="cuda")
            _, tol = _bounded(q[2].double().view(kv, -1, dim), k64, v64, dim ** -0.5, seen, torch.bfloat16, False)
            assert bool(((got[2].double() - reference[first[2] + at[2]].double()).abs().view(tol.shape) <= 2 * tol).all())
        logits = got.float().reshape(3, -1) @ head
        lp, en, ids, tl = _score(qb, logits, [7] * 3, 1.0, 4)
        par, tk = _dev([[-1]] * 3), _dev([[0]] * 3)
        path, n_path, nxt = (torch.empty(3, dtype=torch.int32, device="cuda") for _ in range(3))
        qb.tree_verify(logits.data_ptr(), qb.FP32, 5000, 0, 0, tk.data_ptr(), par.data_ptr(), 0, 3, 1, 5000, 0.0, path.data_ptr(), n_path.data_ptr(), nxt.data_ptr(), _stream())
        torch.cuda.synchronize()
        assert ids[:, 0].tolist() == nxt.tolist()


def test_pages_agree_with_slots(qb):
    """Pages that lie in a contiguous cache's slots: qwen_tree_attention over the slots and qwen_paged_attention over the pages agree
    within both bounds, and rows that qwen_kv_append stores are those that qwen_qk_rope without turning stores."""
    import torch
    g = _gen(12)
    b, kv, cap, dim, page, heads = 3, 2, 512, 128, 32, 6
    k, v = (torch.randn(b, kv, cap, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    slots = qb.KVCache(k.data_ptr(), v.data_ptr(), None, None, k.stride(0), k.stride(1), qb.BF16, b, kv, dim, cap)
    per = kv * cap // page                                  # pages from one sequence to the next
    table = _dev([[s * per + i for i in range(cap // page)] for s in range(b)])
    # page p of sequence s begins at row s * kv * cap + p * page of head 0; a head lies cap rows on
    pages = qb.KVPages(k.data_ptr(), v.data_ptr(), None, None, table.data_ptr(), page * dim, cap * dim, qb.BF16, b * per - cap // page * (kv - 1), b, kv, dim, page, cap // page)
    x = [torch.randn(b * 2, kv * dim, generator=g, device="cuda").bfloat16() for _ in range(2)]
    q = torch.randn(b, heads, dim, generator=g, device="cuda").bfloat16()
    start = _dev([5, 100, 300])
    qb.kv_append(slots, x[0].data_ptr(), x[1].data_ptr(), qb.BF16, kv * dim, 2, start.data_ptr(), 0, _stream())
    after = k.clone(), v.clone()
    qq = torch.empty(b * 2, heads * dim, device="cuda").bfloat16()
    wide = torch.zeros(b * 2, heads * dim, device="cuda").bfloat16()
    # base 1 turns every pair by the position alone; rows of equal values at position 0 .. would turn, so V alone is compared
    pos, sq = _dev([5, 6, 100, 101, 300, 301]), _dev([0, 0, 1, 1, 2, 2])
    v.zero_()
    qb.qk_rope(wide.data_ptr(), x[0].data_ptr(), x[1].data_ptr(), qb.BF16, heads * dim, kv * dim, kv * dim, b * 2, heads, kv, dim, 0, 0, 0, 1e-6, 1e6, pos.data_ptr(),
               qq.data_ptr(), 0, qb.BF16, heads * dim, 0, pages, sq.data_ptr(), _stream())
    for s, p in zip(sq.tolist(), pos.tolist()):
        assert torch.equal(v[s, :, p], after[1][s, :, p])
    v.copy_(after[1])
    lens = _dev([6, 101, 301])
    work = torch.empty(max(qb.paged_attention_workspace(pages, heads), qb.tree_attention_workspace(slots, 1, heads), 16), dtype=torch.uint8, device="cuda")
    outs = [torch.empty(b, heads * dim, device="cuda").bfloat16() for _ in range(2)]
    par = _dev([[-1]] * b)
    qb.paged_attention(pages, q.data_ptr(), outs[0].data_ptr(), qb.BF16, heads * dim, heads * dim, heads, lens.data_ptr(), 0.1, work.data_ptr(), work.numel(), _stream())
    qb.tree_attention(slots, q.data_ptr(), outs[1].data_ptr(), qb.BF16, heads * dim, heads * dim, 1, heads, lens.data_ptr(), par.data_ptr(), 0.1, work.data_ptr(),
                      work.numel(), _stream())
    torch.cuda.synchronize()
    for s, n in enumerate([6, 101, 301]):
        seen = torch.ones(heads // kv, n + 1, dtype=torch.bool, device="cuda")
        want, tol = _bounded(q[s].double().view(kv, -1, dim), k[s, :, :n + 1].double(), v[s, :, :n + 1].double(), 0.1, seen, torch.bfloat16, False)
        for o in outs:
            assert bool(((o[s].double().view(want.shape) - want).abs() <= tol).all())


def _step_buffers(qb, store, seed):
    import torch
    g, rng = _gen(seed), np.random.RandomState(seed)
    b, kv, heads, dim, page, vocab = 4, 2, 6, 64, 16, 3001
    lens = rng.randint(0, 700, b)
    table, pages = _table(rng, [720] * b, page)
    pool = Pool(qb, table, pages, kv, page, dim, store).fill(g)
    s = dict(pool=pool, b=b, kv=kv, heads=heads, dim=dim, vocab=vocab, lens=_dev(lens), seqs=_dev(np.arange(b)))
    for n, w in (("q", heads), ("k", kv), ("v", kv), ("qo", heads), ("out", heads)):
        s[n] = torch.randn(b, w * dim, generator=g, device="cuda").bfloat16()
    s["work"] = torch.empty(qb.paged_attention_workspace(pool.view, heads), dtype=torch.uint8, device="cuda")
    s["logits"], s["tokens"] = torch.randn(b, vocab, generator=g, device="cuda"), _dev(rng.randint(0, vocab, b))
    s["lp"], s["en"] = torch.empty(b, device="cuda"), torch.empty(b, device="cuda")
    s["ids"], s["tl"] = torch.empty(b, 5, dtype=torch.int32, device="cuda"), torch.empty(b, 5, device="cuda")
    s["starts"], s["k_starts"] = _dev([0, 1, 2, 4]), _dev([0, 1, 2, 4])
    s["prompt"] = torch.full((b, heads * dim), 3.0, device="cuda").bfloat16()
    return s


def _step(qb, s, stream):
    """A decode step's calls, and a small prompt's on the same rows."""
    wide, narrow = s["heads"] * s["dim"], s["kv"] * s["dim"]
    qb.qk_rope(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), qb.BF16, wide, narrow, narrow, s["b"], s["heads"], s["kv"], s["dim"], 0, 0, 0, 1e-6, 1e6,
               s["lens"].data_ptr(), s["qo"].data_ptr(), 0, qb.BF16, wide, narrow, s["pool"].view, s["seqs"].data_ptr(), stream)
    qb.paged_attention(s["pool"].view, s["qo"].data_ptr(), s["out"].data_ptr(), qb.BF16, wide, wide, s["heads"], s["lens"].data_ptr(), 0.125, s["work"].data_ptr(),
                       s["work"].numel(), stream)
    qb.prompt_attention(s["qo"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["prompt"].data_ptr(), qb.BF16, wide, narrow, narrow, wide, s["starts"].data_ptr(),
                        s["k_starts"].data_ptr(), 3, s["b"], s["b"], s["heads"], s["kv"], s["dim"], 0.125, stream)
    qb.token_logprobs(s["logits"].data_ptr(), qb.FP32, s["vocab"], s["b"], s["vocab"], s["tokens"].data_ptr(), 1.0, 5, s["lp"].data_ptr(), s["en"].data_ptr(),
                      s["ids"].data_ptr(), s["tl"].data_ptr(), stream)


NAMES = ("qo", "out", "prompt", "lp", "en", "ids", "tl")


@pytest.mark.parametrize("store", ["bf16", "e4m3"])
def test_captured_step_follows_its_inputs(qb, store):
    """A step captured once and replayed with other lengths, pages, starts, rows and logits gives what plain calls give."""
    import torch
    s = _step_buffers(qb, store, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    _step(qb, s, stream.cuda_stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        _step(qb, s, torch.cuda.current_stream().cuda_stream)
    for seed in (2, 3):
        other, plain = _step_buffers(qb, store, seed), _step_buffers(qb, store, seed)
        for n in ("q", "k", "v", "lens", "logits", "tokens"):
            s[n].copy_(other[n])
        s["starts"].copy_(_dev([0, 3, 3, 4]))
        s["k_starts"].copy_(_dev([0, 3, 3, 4]))
        plain["starts"], plain["k_starts"] = s["starts"], s["k_starts"]
        s["pool"].table_dev.copy_(other["pool"].table_dev)
        for n in ("k_all", "v_all", "ks_all", "vs_all"):
            if getattr(s["pool"], n) is not None:
                getattr(s["pool"], n).copy_(getattr(other["pool"], n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _step(qb, plain, _stream())
        torch.cuda.synchronize()
        for n in NAMES:
            assert torch.equal(s[n], plain[n]), n
        for a, b in zip(s["pool"].raw(), plain["pool"].raw()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("store", ["bf16", "int8"])
def test_captured_clusters_follow_their_inputs(qb, store):
    """Attention by clusters (few sequences, no workspace), captured once and replayed with other lengths, tables and queries."""
    import torch
    rng, g = np.random.RandomState(21), _gen(21)
    b, kv, heads, dim, page, most = 2, 4, 12, 128, 16, 2000
    table, pages = _table(rng, [most] * b, page)
    pool = Pool(qb, table, pages, kv, page, dim, store).fill(g)
    assert qb.paged_attention_workspace(pool.view, heads) == 0
    q, out, lens = torch.zeros(b, heads * dim, device="cuda").bfloat16(), torch.empty(b, heads * dim, device="cuda").bfloat16(), _dev([0, 0])
    call = lambda o, st: qb.paged_attention(pool.view, q.data_ptr(), o.data_ptr(), qb.BF16, heads * dim, heads * dim, heads, lens.data_ptr(), 0.09, 0, 0, st)  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    call(out, stream.cuda_stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(out, torch.cuda.current_stream().cuda_stream)
    for n in ([1999, 3], [-1, 700], [63, 1024], [2 ** 30, 0]):
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        lens.copy_(_dev(n))
        pool.table = table[:, rng.permutation(table.shape[1])]
        pool.table_dev.copy_(_dev(pool.table))
        out.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(b, heads, dim), _check_paged(qb, pool, q.view(b, heads, dim), n, 0.09))


def test_two_streams_and_repeats(qb):
    """Steps on two streams at once, each with its own workspace, repeated: always the same bits."""
    import torch
    sets = [_step_buffers(qb, "bf16", 5), _step_buffers(qb, "int8", 6)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    want = []
    for s in sets:
        _step(qb, s, _stream())
        torch.cuda.synchronize()
        want.append({n: s[n].clone() for n in NAMES})
    for _ in range(5):
        for s in sets:
            for n in NAMES:
                s[n].fill_(1)
            s["prompt"].fill_(3)
        torch.cuda.synchronize()
        for _ in range(3):
            for s, st in zip(sets, streams):
                _step(qb, s, st.cuda_stream)
        torch.cuda.synchronize()
        for s, w in zip(sets, want):
            for n in NAMES:
                assert torch.equal(s[n], w[n]), n


def test_refusals_on_the_device(qb):
    """Host memory, too small a workspace: refused with a message, and the next call works."""
    import torch
    s = _step_buffers(qb, "bf16", 7)
    wide, narrow = s["heads"] * s["dim"], s["kv"] * s["dim"]
    for bad in (torch.zeros(4096, dtype=torch.int32).data_ptr(), torch.zeros(4096, dtype=torch.int32).pin_memory().data_ptr()):
        for f in (lambda: qb.qk_rope(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), qb.BF16, wide, narrow, narrow, s["b"], s["heads"], s["kv"], s["dim"], 0, 0, 0,
                                     1e-6, 1e6, bad, s["qo"].data_ptr(), 0, qb.BF16, wide, narrow, s["pool"].view, s["seqs"].data_ptr()),
                  lambda: qb.paged_attention(s["pool"].view, s["q"].data_ptr(), s["out"].data_ptr(), qb.BF16, wide, wide, s["heads"], bad, 0.1, s["work"].data_ptr(),
                                             s["work"].numel()),
                  lambda: qb.prompt_attention(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), qb.BF16, wide, narrow, narrow, wide, bad, 0, 1,
                                              s["b"], s["b"], s["heads"], s["kv"], s["dim"], 0.1),
                  lambda: qb.token_logprobs(s["logits"].data_ptr(), qb.FP32, s["vocab"], s["b"], s["vocab"], bad, 1.0, 0, s["lp"].data_ptr(), 0, 0, 0)):
            with pytest.raises(qb.QwenError) as e:
                f()
            assert e.value.code == -1 and "device memory" in str(e.value)
    assert s["work"].numel() > 0
    with pytest.raises(qb.QwenError) as e:
        qb.paged_attention(s["pool"].view, s["q"].data_ptr(), s["out"].data_ptr(), qb.BF16, wide, wide, s["heads"], s["lens"].data_ptr(), 0.1, s["work"].data_ptr(),
                           s["work"].numel() - 1)
    assert e.value.code == -1 and "workspace" in str(e.value)
    _step(qb, s, _stream())
    torch.cuda.synchronize()
    assert bool(s["out"].isfinite().all())
