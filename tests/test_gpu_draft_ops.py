"""The drafted-token operators (qwen_kv_append, qwen_kv_read, qwen_kv_keep,
qwen_tree_attention, qwen_tree_verify) against plain implementations in 64 bits:
codes, moved rows, paths and tokens exactly, attention within the roundings that
its documentation names."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOP = {"e4m3": 448.0, "int8": 127.0}
DIRTY = 0x5A      # what unwritten bytes of caches and outputs hold


def _types(qb):
    import torch
    return {"bf16": (qb.BF16, torch.bfloat16), "fp16": (qb.FP16, torch.float16), "fp32": (qb.FP32, torch.float32),
            "e4m3": (qb.E4M3, torch.float8_e4m3fn), "int8": (qb.INT8, torch.int8)}


class Cache:
    """A cache [b][kv][cap][dim], optionally with room between heads and sequences, and its view."""

    def __init__(self, qb, b, kv, cap, dim, store, room=0):
        import torch
        self.kind, self.dtype = _types(qb)[store]
        self.store, self.b, self.kv, self.cap, self.dim = store, b, kv, cap, dim
        heads = kv + (1 if room else 0)
        full = lambda *s: torch.full((*s, self.dtype.itemsize), DIRTY, dtype=torch.uint8, device="cuda").view(self.dtype)[..., 0]  # noqa: E731
        self.k_all, self.v_all = full(b, heads, cap + room, dim), full(b, heads, cap + room, dim)
        self.k, self.v = self.k_all[:, :kv, :cap], self.v_all[:, :kv, :cap]
        self.ks_all = self.vs_all = self.ks = self.vs = None
        if store in TOP:
            self.ks_all = torch.full((b, heads, cap + room), -7.0, device="cuda")
            self.vs_all = torch.full((b, heads, cap + room), -7.0, device="cuda")
            self.ks, self.vs = self.ks_all[:, :kv, :cap], self.vs_all[:, :kv, :cap]
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.view = qb.KVCache(p(self.k_all), p(self.v_all), p(self.ks_all), p(self.vs_all), self.k_all.stride(0), self.k_all.stride(1), self.kind,
                               b, kv, dim, cap)

    def fill(self, g, spread=1.0):
        """Rows of normal values, quantised plainly for the 8-bit types."""
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

    def values(self):
        """K and V in 64 bits."""
        out = []
        for x, s in ((self.k, self.ks), (self.v, self.vs)):
            y = x.float().double()
            out.append(y if s is None else y * s[..., None].double())
        return out

    def raw(self):
        import torch
        return [t.clone().view(torch.uint8) if t.dtype.itemsize == 1 else t.clone().view(torch.int16) if t.dtype.itemsize == 2
                else t.clone().view(torch.int32) for t in (self.k_all, self.v_all, self.ks_all, self.vs_all) if t is not None]


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------------------
# rows in and out
# ---------------------------------------------------------------------------
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


def _rows(g, shape, dtype, kind):
    import torch
    x = torch.randn(shape, generator=g, device="cuda")
    if kind == "ties":      # small whole numbers: many quotients lie half way between two codes
        x = torch.randint(-96, 97, shape, generator=g, device="cuda").float()
    elif kind == "wide":    # magnitudes from the smallest to the largest of the type
        x = x * torch.exp2(torch.randint(-20 if dtype == torch.float16 else -140, 14 if dtype == torch.float16 else 125, shape[:-1],
                                         generator=g, device="cuda").float())[..., None]
    return x.to(dtype)


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("src", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind,b,t,kv,dim", [("normal", 3, 37, 2, 128), ("ties", 2, 129, 3, 64), ("wide", 2, 65, 1, 128), ("normal", 5, 1, 8, 64)])
def test_append_codes_are_the_nearest(qb, store, src, kind, b, t, kv, dim):
    """Codes and scales equal the 64-bit definition's; everything else of the cache stays as it was."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t)
    kind_src, dtype = _types(qb)[src]
    c = Cache(qb, b, kv, t + 9, dim, store, room=3)
    before = c.raw()
    x = [_rows(g, (b, t, kv * dim + 16), dtype, kind) for _ in range(2)]           # rows with room behind them
    start = np.array([(5 * r) % 10 for r in range(b)], np.int32)
    counts = np.array([t if r == 0 else (t * r) // b for r in range(b)], np.int32)
    st, ct = _dev(start), _dev(counts)
    qb.kv_append(c.view, x[0].data_ptr(), x[1].data_ptr(), kind_src, kv * dim + 16, t, st.data_ptr(), ct.data_ptr(), _stream())
    after = c.raw()
    for i, (rows, got, scale) in enumerate(((x[0], c.k, c.ks), (x[1], c.v, c.vs))):
        whole = (c.k_all, c.v_all)[i].clone().view(torch.uint8)
        for r in range(b):
            n, s = int(counts[r]), int(start[r])
            want, a = _codes64(rows[r, :n, :kv * dim].view(n, kv, dim).double().transpose(0, 1), store)
            assert torch.equal(got[r, :, s:s + n].float().double(), want), (store, src, kind, r)
            assert torch.equal(scale[r, :, s:s + n], a[..., 0].float())
            whole[r, :kv, s:s + n] = DIRTY
            after[2 + i].view(torch.float32)[r, :kv, s:s + n] = -7.0
        assert bool((whole == DIRTY).all())
        assert torch.equal(after[2 + i], before[2 + i])


@pytest.mark.parametrize("store,src,dim,t", [("e4m3", "bf16", 128, 5501), ("int8", "fp16", 128, 5469), ("int8", "bf16", 64, 10977), ("e4m3", "fp32", 64, 10923),
                                             ("bf16", "bf16", 128, 5501)])
def test_append_many_rows(qb, store, src, dim, t):
    """Prompts of several sequences, none of a whole number of blocks: every row, and nothing beside them."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t)
    kind_src, dtype = _types(qb)[src]
    b, kv = 3, 8
    c = Cache(qb, b, kv, t + 2, dim, store, room=1)
    x = [_rows(g, (b, t, kv * dim), dtype, "ties" if store == "e4m3" else "normal") for _ in range(2)]
    start, counts = np.array([2, 0, 5], np.int32), np.array([t, t - 1001, t], np.int32)     # the last sequence runs out of the cache
    st, ct = _dev(start), _dev(counts)
    qb.kv_append(c.view, x[0].data_ptr(), x[1].data_ptr(), kind_src, kv * dim, t, st.data_ptr(), ct.data_ptr(), _stream())
    for rows, got, all_, scale, sc_all in ((x[0], c.k, c.k_all, c.ks, c.ks_all), (x[1], c.v, c.v_all, c.vs, c.vs_all)):
        for r in range(b):
            s, n = int(start[r]), min(int(counts[r]), c.cap - int(start[r]))
            y = rows[r, :n].view(n, kv, dim).transpose(0, 1)
            if scale is None:
                assert torch.equal(got[r, :, s:s + n], y.to(c.dtype))
            else:
                want, a = _codes64(y.double(), store)
                assert torch.equal(got[r, :, s:s + n].float(), want.float()) and torch.equal(scale[r, :, s:s + n], a[..., 0].float())
                sc_all[r, :kv, s:s + n] = -7.0
            all_.view(torch.uint8)[r, :kv, s:s + n] = DIRTY
        assert bool((all_.view(torch.uint8) == DIRTY).all()) and (scale is None or bool((sc_all == -7.0).all()))


@pytest.mark.parametrize("store", ["e4m3", "int8", "bf16", "fp16"])
@pytest.mark.parametrize("dst", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("b,t,kv,dim", [(3, 41, 2, 128), (4, 1, 3, 64)])
def test_read_is_code_times_scale(qb, store, dst, b, t, kv, dim):
    import torch
    g = torch.Generator(device="cuda").manual_seed(7)
    kind_dst, dtype = _types(qb)[dst]
    c = Cache(qb, b, kv, t + 6, dim, store, room=2).fill(g)
    start = np.array([0, 6, 3, -1][:b], np.int32)
    counts = np.array([t, max(t - 3, 1), 0, t][:b], np.int32)
    ld = kv * dim + 8
    out = [torch.full((b, t, ld), 3.0, dtype=dtype, device="cuda") for _ in range(2)]
    st, ct = _dev(start), _dev(counts)
    qb.kv_read(c.view, out[0].data_ptr(), out[1].data_ptr(), kind_dst, ld, t, st.data_ptr(), ct.data_ptr(), _stream())
    for got, x, s in ((out[0], c.k, c.ks), (out[1], c.v, c.vs)):
        want = torch.full((b, t, ld), 3.0, dtype=dtype, device="cuda")
        for r in range(b):
            if start[r] < 0:
                continue
            a, n = int(start[r]), int(counts[r])
            y = x[r, :, a:a + n].float()
            y = y if s is None else y * s[r, :, a:a + n, None]
            want[r, :n, :kv * dim] = y.to(dtype).transpose(0, 1).reshape(n, kv * dim)
        assert torch.equal(got, want)


def test_append_special_rows(qb):
    """Zero, tiny and non-finite rows; positions outside the cache; idle sequences."""
    import torch
    for store in ("e4m3", "int8"):
        c = Cache(qb, 3, 1, 4, 64, store)
        x = torch.zeros(3, 4, 64, device="cuda")
        x[0, 1] = 1e-30
        x[0, 2, 5], x[0, 2, 6] = float("inf"), 1.0
        x[0, 3, 9] = float("nan")
        x[1] = torch.arange(256, device="cuda").view(4, 64) * 1e36
        start = _dev(np.array([0, 2, -5], np.int32))
        qb.kv_append(c.view, x.data_ptr(), x.data_ptr(), qb.FP32, 64, 4, start.data_ptr(), 0, _stream())
        out = torch.full((3, 4, 64), 9.0, device="cuda")
        rest = torch.empty_like(out)
        qb.kv_read(c.view, out.data_ptr(), rest.data_ptr(), qb.FP32, 64, 4, start.data_ptr(), 0, _stream())
        assert bool((out[0, 0] == 0).all()) and bool((out[0, 1].abs() <= 2.0 ** -60).all())
        assert bool(out[0, 2].isnan().all()) and bool(out[0, 3].isnan().all())
        step = 2.0 ** -4 if store == "e4m3" else 0.5 / 127            # half a step: relative, or of the row's largest
        assert bool(((out[1, :2] - x[1, :2]).abs() <= step * (x[1, :2] if store == "e4m3" else x[1, :2].amax(-1, keepdim=True)) * 1.001
                     + x[1, :2].amax(-1, keepdim=True) * 2.0 ** -10 / 448 * 1.001).all())
        assert bool((out[1, 2:] == 9).all()) and bool((out[2] == 9).all())     # positions 4, 5 and the idle sequence
        assert bool((c.ks[1, :, :2] == -7).all()) and bool((c.ks[2] == -7).all())


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("b,t,kv,dim", [(4, 64, 3, 128), (3, 5, 2, 64), (2, 1, 1, 128), (3, 17, 1, 64)])
def test_keep_moves_rows(qb, store, b, t, kv, dim):
    """Ascending paths, any order, repeats, entries out of range, idle sequences, a cache that ends inside the tree."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(11)
    rng = np.random.RandomState(t)
    for mode in range(4):
        c = Cache(qb, b, kv, t + 5, dim, store, room=1).fill(g)
        path = np.full((b, t), -1, np.int32)
        count = rng.randint(0, t + 1, b).astype(np.int32)
        start = rng.randint(0, 6, b).astype(np.int32)
        for r in range(b):
            p = np.sort(rng.choice(t, count[r], replace=False)) if mode == 0 else rng.randint(0, t, count[r])
            path[r, :count[r]] = p
        if mode == 2:
            path[rng.rand(b, t) < 0.3] = t + 3
            start[0] = -1
            count[-1] = t + 40       # more than there are: the row's t entries
        if mode == 3:
            start[:] = 5 + t // 2    # the tree's later positions lie outside
        before = [x.clone() for x in (c.k_all, c.v_all, c.ks_all, c.vs_all) if x is not None]
        st, ph, ct = _dev(start), _dev(path), _dev(count)
        qb.kv_keep(c.view, st.data_ptr(), ph.data_ptr(), ct.data_ptr(), t, _stream())
        for was, now in zip(before, [x for x in (c.k_all, c.v_all, c.ks_all, c.vs_all) if x is not None]):
            want = was.clone().view(torch.uint8) if was.dtype.itemsize == 1 else was.clone()
            src = was.view(torch.uint8) if was.dtype.itemsize == 1 else was
            for r in range(b):
                s = int(start[r])
                if s < 0:
                    continue
                for i in range(min(int(count[r]), t)):
                    p = int(path[r, i])
                    if 0 <= p < t and s + p < c.cap and s + i < c.cap:
                        want[r, :kv, s + i] = src[r, :kv, s + p]
            assert torch.equal(now.view(torch.uint8) if now.dtype.itemsize == 1 else now, want), mode


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _sees(parents, length, cap):
    """Which nodes each node sees, as sets (None: absent)."""
    out = []
    for i, p in enumerate(parents):
        if length < 0 or length + i >= cap or p < -1 or p >= i or (p >= 0 and out[p] is None):
            out.append(None)
        else:
            out.append(({i} | out[p]) if p >= 0 else {i})
    return out


def _attention64(c, q, lens, parents, scale):
    """The definition in 64 bits, and a bound on a kernel's error: the weights' and the output's roundings
    (half a step of the product's 16-bit type each), fp32 scores, and fp16's smallest steps for 8-bit values."""
    import torch
    b, t, heads, dim = q.shape
    group = heads // c.kv
    k64, v64 = c.values()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    half = torch.finfo(q.dtype).eps / 2
    half_p = torch.finfo(torch.float16).eps / 2 if c.store in TOP else half
    for r in range(b):
        seen = _sees(parents[r].tolist(), int(lens[r]), c.cap)
        for i, up in enumerate(seen):
            if up is None:
                continue
            at = list(range(int(lens[r]))) + [int(lens[r]) + j for j in sorted(up)]
            k, v = k64[r][:, at], v64[r][:, at]
            x = q[r, i].double().view(c.kv, group, dim)
            s = torch.einsum("hgd,hkd->hgk", x, k) * scale
            w = torch.softmax(s, -1)
            o = torch.einsum("hgk,hkd->hgd", w, v)
            av = torch.einsum("hgk,hkd->hgd", w, v.abs())
            size = (torch.einsum("hgd,hkd->hgk", x.abs(), k.abs()) * abs(scale)).amax(-1, keepdim=True)
            # a weight's relative error: its 16-bit rounding (8-bit rows: of weight times scale), the fp32 products and
            # sums behind the score (dim + 8 roundings of at most `size`), exp2's argument and result
            rel = half_p + 2 * (dim + 8) * 2.0 ** -24 * size + 2.0 ** -20
            vmax = v.abs().amax(1)[:, None]
            o_tol = rel * av + (2.0 ** -23 * len(at) * vmax if c.store in TOP or q.dtype == torch.float16 else 0)
            out[r, i] = o.reshape(heads, dim)
            tol[r, i] = (o_tol * (1 + half) + half * o.abs() + 2.0 ** -24 * (q.dtype == torch.float16)).reshape(heads, dim)
    return out, tol


def _attend(qb, c, q, lens, parents, scale, ldq=None, ldo=None, stream=None):
    import torch
    b, t, heads, dim = q.shape
    ldq, ldo = ldq or heads * dim, ldo or heads * dim
    kind = qb.BF16 if q.dtype == torch.bfloat16 else qb.FP16
    qs = torch.full((b, t, ldq), float("nan"), dtype=q.dtype, device="cuda")
    qs[..., :heads * dim] = q.reshape(b, t, heads * dim)
    out = torch.full((b, t, ldo), 5.0, dtype=q.dtype, device="cuda")
    work = torch.full((qb.tree_attention_workspace(c.view, t, heads),), 0xFF, dtype=torch.uint8, device="cuda")   # NaN
    ln, pr = _dev(np.asarray(lens, np.int32)), _dev(np.asarray(parents, np.int32))
    qb.tree_attention(c.view, qs.data_ptr(), out.data_ptr(), kind, ldq, ldo, t, heads, ln.data_ptr(), pr.data_ptr(), scale, work.data_ptr(),
                      work.numel(), _stream() if stream is None else stream)
    torch.cuda.synchronize()
    assert bool((out[..., heads * dim:] == 5).all())
    return out[..., :heads * dim].reshape(b, t, heads, dim)


def _tree(rng, b, t, absent=False):
    par = np.empty((b, t), np.int32)
    for i in range(t):
        par[:, i] = -1 if i == 0 else rng.randint(-1 if i % 5 == 0 else max(0, i - 4), i, b)
    if absent:
        par[rng.rand(b, t) < 0.15] = -3
        par[rng.rand(b, t) < 0.05] = 64
        par[0, t // 2:] = -2
    return par


def _check_attention(qb, c, q, lens, parents, scale, **kw):
    import torch
    got = _attend(qb, c, q, lens, parents, scale, **kw).double()
    want, tol = _attention64(c, q, lens, parents, scale)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() / tol.clamp_min(1e-30))[bad].max()), bad.nonzero()[:4].tolist())
    return got


@pytest.mark.parametrize("store", ["16", "e4m3", "int8"])
@pytest.mark.parametrize("qt", ["bf16", "fp16"])
@pytest.mark.parametrize("t,group,dim", [(1, 1, 128), (1, 2, 64), (7, 2, 128), (5, 3, 64), (16, 4, 128), (64, 2, 128), (64, 1, 64), (33, 8, 128)])
def test_attention_ragged_batches(qb, store, qt, t, group, dim):
    """Lengths from none to several tiles, on both sides of a tile's end, with trees and absent nodes."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t * 7 + group)
    rng = np.random.RandomState(t)
    lens = [0, 1, 63, 64, 65, 127, 200, 331 - t]
    kv = 2 if group < 8 else 1
    c = Cache(qb, len(lens), kv, 331, dim, qt if store == "16" else store, room=5).fill(g)
    q = torch.randn(len(lens), t, kv * group, dim, generator=g, device="cuda").to(_types(qb)[qt][1])
    _check_attention(qb, c, q, lens, _tree(rng, len(lens), t, absent=t > 4), 1 / math.sqrt(dim), ldq=kv * group * dim + 24, ldo=kv * group * dim + 8)


@pytest.mark.parametrize("store,t,group,kv", [("bf16", 1, 2, 8), ("bf16", 64, 2, 2), ("bf16", 64, 8, 1), ("e4m3", 8, 2, 8), ("int8", 4, 4, 1), ("e4m3", 64, 2, 1)])
def test_attention_long(qb, store, t, group, kv):
    """One long sequence: the key axis split over all SMs and joined."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    c = Cache(qb, 1, kv, 8192, 128, store).fill(g)
    q = torch.randn(1, t, kv * group, 128, generator=g, device="cuda").to(torch.bfloat16)
    _check_attention(qb, c, q, [8192 - t], _tree(np.random.RandomState(1), 1, t), 1 / math.sqrt(128))


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_attention_absent_and_outside(qb, store):
    """Idle sequences (negative and too large lengths) give 0; nodes past the capacity are absent."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    t, cap = 6, 70
    c = Cache(qb, 6, 2, cap, 128, store, room=2).fill(g)
    q = torch.randn(6, t, 4, 128, generator=g, device="cuda").to(torch.bfloat16)
    lens = [-1, cap, cap - 3, 2 ** 31 - 1, -2 ** 31, 10]
    par = np.tile(np.arange(-1, t - 1, dtype=np.int32), (6, 1))
    got = _check_attention(qb, c, q, lens, par, 0.1)
    for r in (0, 1, 3, 4):
        assert bool((got[r] == 0).all())
    assert bool((got[2, 3:] == 0).all()) and bool((got[2, :3] != 0).any())
    par[:] = -2                                  # nothing is present at all
    assert bool((_attend(qb, c, q, lens, par, 0.1) == 0).all())


@pytest.mark.parametrize("store", ["bf16", "fp16", "e4m3", "int8"])
@pytest.mark.parametrize("t,length", [(2, 0), (5, 17), (64, 100), (64, 64)])
def test_attention_unseen_values_do_not_matter(qb, store, t, length):
    """NaN and infinities behind the sequence and in branches that a node does not see change nothing; in one that it sees, they show."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(length)
    dim, cap = 64, length + t + 30
    c = Cache(qb, 2, 2, cap, dim, store).fill(g)
    q = torch.randn(2, t, 4, dim, generator=g, device="cuda").to(torch.float16 if store == "fp16" else torch.bfloat16)
    par = np.zeros((2, t), np.int32)
    par[:, 0] = -1
    par[:, 1:] = 0                               # siblings below one root
    lens = [length, length]
    clean = _check_attention(qb, c, q, lens, par, 0.125)
    bad = [length + i for i in range(1, t) if i % 2 == 0] + list(range(length + t, cap))
    for x, s in ((c.k, c.ks), (c.v, c.vs)):
        if s is not None:
            s[:, :, bad] = float("nan")
            s[:, :, length + t] = float("inf")
        if store == "e4m3":
            x[0].view(torch.uint8)[:, bad] = 0x7F
        elif store != "int8":
            x[0][:, bad] = float("nan")
            x[1][:, bad, ::3] = float("inf")
    got = _attend(qb, c, q, lens, par, 0.125).double()
    good = [i for i in range(t) if i == 0 or i % 2]
    assert torch.equal(got[:, good], clean[:, good])
    for i in range(2, t, 2):
        assert not bool(got[:, i].isfinite().all())


@pytest.mark.parametrize("store", ["bf16", "int8"])
@pytest.mark.parametrize("t,cap", [(6, 200), (6, 1500), (40, 300), (40, 1500)])
def test_attention_any_negative_length_is_idle(qb, store, t, cap):
    """Lengths down to the smallest number: their sequences' rows are 0, the others right."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t)
    lens = [cap - t, -1, -2 ** 31, -2 ** 31 + 1, -2 ** 31 + 70, 33]
    c = Cache(qb, len(lens), 2, cap, 128, store).fill(g)
    q = torch.randn(len(lens), t, 4, 128, generator=g, device="cuda").to(torch.bfloat16)
    got = _check_attention(qb, c, q, lens, _tree(np.random.RandomState(t), len(lens), t), 0.1)
    assert bool((got[1:5] == 0).all()) and bool((got[[0, 5]] != 0).any())


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("t,group,dim,length,cap", [(6, 2, 128, 20, 60), (6, 2, 64, 0, 60), (12, 2, 64, 117, 300), (24, 1, 128, 50, 150), (40, 1, 128, 100, 300),
                                                    (64, 2, 64, 33, 200), (64, 8, 128, 90, 160), (6, 2, 128, 1270, 1400), (28, 1, 64, 1273, 1400), (64, 1, 128, 1215, 1400),
                                                    (64, 3, 64, 1280, 1400)])
def test_attention_unseen_scales_do_not_matter(qb, store, t, group, dim, length, cap):
    """Scales of any size at positions that a node does not see (another branch's, an absent node's, those behind a short count)
    leave its result as it is, bit for bit; the nodes that see such rows are right as well."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t + length)
    b, kv = 3, 2
    clean = Cache(qb, b, kv, cap, dim, store).fill(g)
    q = torch.randn(b, t, kv * group, dim, generator=g, device="cuda").to(torch.bfloat16)
    here = t - t // 4                            # nodes from here on are absent
    par = np.full((b, t), -2, np.int32)
    par[:, 0] = -1
    for i in range(1, here):                     # two branches: 0, 1, 3, 5, .. and 0, 2, 4, ..
        par[:, i] = max(0, i - 2)
    lens = [length, max(length - 9, 0), length // 2]
    want = _attend(qb, clean, q, lens, par, dim ** -0.5)
    assert bool(want[:, :here].isfinite().all()) and bool((want[:, :here] != 0).any(-1).all())

    def poisoned(nodes, value, behind):
        c = Cache(qb, b, kv, cap, dim, store)
        for x, y in ((c.k, clean.k), (c.v, clean.v)):
            x.view(torch.uint8).copy_(y.view(torch.uint8))
        for x, y in ((c.ks, clean.ks), (c.vs, clean.vs)):
            x.copy_(y)
            for r in range(b):
                at = [lens[r] + i for i in nodes if lens[r] + i < cap]
                x[r, :, at] = value
                if behind:
                    x[r, :, lens[r] + t:] = value
        return c

    for value in (1e-30, 1e5, -1e9, 1e30, torch.finfo(torch.float32).max):
        got = _attend(qb, poisoned(range(here, t), value, True), q, lens, par, dim ** -0.5)
        assert torch.equal(got, want), value
        got = _attend(qb, poisoned(range(2, t, 2), value, False), q, lens, par, dim ** -0.5)
        odd = [0] + list(range(1, here, 2))
        assert torch.equal(got[:, odd], want[:, odd]), value
    for value in (1e-20, 10.0, 60.0, 3e3, 1e18): # rows that see them: large values, but an ordinary score
        c = poisoned(range(2, t, 2), value, True)
        c.ks.copy_(clean.ks)
        got = _attend(qb, c, q, lens, par, dim ** -0.5).double()
        want64, tol = _attention64(c, q, lens, par, dim ** -0.5)
        codes = c.v.float().double().abs()
        for r in range(b):                       # Weight times scale is fp16 in a unit of at most twice the largest seen scale: half of its
            for i in range(here):                # smallest step is 2^-25 of that, for each key's code; the sum of the weights is at least 1.
                at = list(range(lens[r])) + [lens[r] + j for j in sorted(_sees(par[r].tolist(), lens[r], cap)[i])]
                low = 2.0 ** -24 * c.vs[r][:, at].double().amax(1)[:, None] * codes[r][:, at].sum(1)
                tol[r, i] += low.repeat_interleave(group, 0)
        assert bool(((got - want64).abs() <= tol).all()), value


@pytest.mark.parametrize("store", ["e4m3", "int8"])
@pytest.mark.parametrize("t,group,dim,cap,low,high", [(3, 2, 128, 300, -60, 115), (3, 2, 128, 1400, -60, 115), (7, 4, 64, 300, 90, 115), (12, 2, 128, 1400, -60, 60),
                                                      (40, 1, 128, 300, -30, 90), (40, 2, 64, 1400, 60, 90)])
def test_attention_value_scales_of_any_size(qb, store, t, group, dim, cap, low, high):
    """Value rows between 2^low and 2^high: the small ones vanish beside the large, and every key counts in the sum of the weights."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t + high)
    c = Cache(qb, 2, 2, cap, dim, store).fill(g)
    c.vs *= torch.exp2(torch.randint(low, high + 1, c.vs.shape, generator=g, device="cuda").float())
    q = torch.randn(2, t, 2 * group, dim, generator=g, device="cuda").to(torch.bfloat16)
    lens, par = [cap - t, cap // 3], _tree(np.random.RandomState(t), 2, t)
    got = _attend(qb, c, q, lens, par, dim ** -0.5).double()
    want, tol = _attention64(c, q, lens, par, dim ** -0.5)
    codes = c.v.float().double().abs()
    for r in range(2):                           # fp16's smallest steps, as above: 2^-24 of the largest seen scale for each key's code
        for i, up in enumerate(_sees(par[r].tolist(), lens[r], cap)):
            if up is not None:
                at = list(range(lens[r])) + [lens[r] + j for j in sorted(up)]
                low_bits = 2.0 ** -24 * c.vs[r][:, at].double().amax(1)[:, None] * codes[r][:, at].sum(1)
                tol[r, i] += low_bits.repeat_interleave(group, 0)
    assert bool(((got - want).abs() <= tol).all())


def test_attention_infinity_in_a_seen_branch(qb):
    """A V row with one infinity: that dim of the nodes that see it becomes infinite, nothing else changes."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    c = Cache(qb, 1, 1, 40, 128, "bf16").fill(g)
    q = torch.randn(1, 3, 2, 128, generator=g, device="cuda").to(torch.bfloat16)
    par = np.array([[-1, 0, 0]], np.int32)
    clean = _attend(qb, c, q, [20], par, 0.1)
    c.v[0, 0, 22, 77] = float("-inf")
    got = _attend(qb, c, q, [20], par, 0.1)
    want = clean.clone()
    want[0, 2, :, 77] = float("-inf")
    assert torch.equal(got, want)


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_attention_extreme_values(qb, store):
    """Scores far apart, negative scale, large and small rows: softmax stays within its roundings."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(9)
    c = Cache(qb, 2, 2, 300, 128, store).fill(g, spread=4.0)
    if store != "bf16":
        c.vs[:, :, ::7] *= 1e4
        c.ks[:, :, 5] *= 30
        c.vs[:, :, 3::11] *= 1e-6
    else:
        c.v[:, :, ::7] *= 1e4
    q = torch.randn(2, 9, 4, 128, generator=g, device="cuda").to(torch.bfloat16)
    q[0, 3] *= 1e-3
    q[1, 4] *= 64
    q[0, 1] = 0
    for scale in (0.3, -0.05, 0.0):
        _check_attention(qb, c, q, [250, 291], _tree(np.random.RandomState(2), 2, 9), scale)


@pytest.mark.parametrize("scale", [0.0, 2e-38, -2e-38])
@pytest.mark.parametrize("t,group", [(1, 2), (40, 2)])
def test_attention_scales_at_the_low_end(qb, scale, t, group):
    """Products of queries and keys up to 10^38, which a scale near the smallest fp32 number, or of 0, brings back."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t)
    c = Cache(qb, 2, 2, 331, 128, "bf16").fill(g)
    c.k *= 1e18
    q = (torch.randn(2, t, 2 * group, 128, generator=g, device="cuda") * 1e18).bfloat16()
    _check_attention(qb, c, q, [280, 7], _tree(np.random.RandomState(t), 2, t), scale)


def test_attention_many_sequences(qb):
    """More sequences than the shares' search takes in one step, most of them short."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    b, t = 333, 3
    c = Cache(qb, b, 2, 140, 64, "bf16").fill(g)
    q = torch.randn(b, t, 6, 64, generator=g, device="cuda").to(torch.bfloat16)
    rng = np.random.RandomState(8)
    lens = np.where(rng.rand(b) < 0.2, rng.randint(0, 138, b), rng.randint(-1, 3, b))
    _check_attention(qb, c, q, lens, _tree(rng, b, t, absent=True), 0.125)


@pytest.mark.parametrize("store", ["16", "e4m3", "int8"])
@pytest.mark.parametrize("t,group,dim,qt", [(1, 1, 64, "bf16"), (1, 2, 128, "fp16"), (5, 3, 64, "bf16"), (16, 2, 128, "bf16"), (11, 4, 128, "fp16"), (64, 2, 128, "bf16"),
                                            (64, 1, 64, "fp16"), (64, 7, 128, "bf16"), (33, 16, 64, "fp16")])
def test_attention_shared_out(qb, store, t, group, dim, qt):
    """Caches long enough that the sequences' tiles are shared out over all SMs: idle, empty, short and long sequences among each
    other, lengths on both sides of a tile's end, several blocks of rows, absent nodes, nodes past the capacity."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(t * 7 + group)
    cap = 1400
    lens = [0, 1400 - t, -1, 1, 511, 512, 513, cap + 5, 640, 1100, 127, 128, 129, cap - 1, 3, 1024 - t]
    c = Cache(qb, len(lens), 2, cap, dim, qt if store == "16" else store, room=5).fill(g)
    assert qb.tree_attention_workspace(c.view, t, 2 * group) > 0
    q = torch.randn(len(lens), t, 2 * group, dim, generator=g, device="cuda").to(_types(qb)[qt][1])
    par = _tree(np.random.RandomState(t), len(lens), t, absent=t > 4)
    _check_attention(qb, c, q, lens, par, 1 / math.sqrt(dim), ldq=2 * group * dim + 24, ldo=2 * group * dim + 8)


@pytest.mark.parametrize("b,t,group,cap,dim,store", [(333, 3, 3, 1100, 64, "bf16"), (129, 1, 2, 1090, 128, "e4m3"), (150, 40, 1, 1030, 64, "int8"),
                                                     (131, 9, 4, 1025, 128, "bf16"), (1, 64, 300, 1100, 64, "bf16"), (2, 64, 301, 1030, 64, "e4m3")])
def test_attention_shared_out_widely(qb, b, t, group, cap, dim, store):
    """More sequences than a block keeps the lengths of, most of them short; more blocks of rows than SMs."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    c = Cache(qb, b, 1, cap, dim, store).fill(g)
    assert qb.tree_attention_workspace(c.view, t, group) > 0
    q = torch.randn(b, t, group, dim, generator=g, device="cuda").to(torch.bfloat16)
    rng = np.random.RandomState(8)
    lens = np.where(rng.rand(b) < 0.2, rng.randint(0, cap - 1, b), rng.randint(-1, 3, b))
    if b < 3:
        lens[:] = cap - t - 3
    _check_attention(qb, c, q, lens, _tree(rng, b, t, absent=True), 0.125)


@pytest.mark.parametrize("b,t,group,cap,dim,store", [(460, 1, 2, 1024, 64, "bf16"), (450, 3, 2, 1000, 128, "int8"), (310, 4, 8, 1024, 128, "e4m3"), (150, 33, 1, 1024, 128, "bf16"),
                                                     (150, 20, 2, 1000, 64, "e4m3")])
def test_attention_without_workspace(qb, b, t, group, cap, dim, store):
    """As many short caches as there are blocks: each is attended to by one, and no workspace is needed."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    c = Cache(qb, b, 1, cap, dim, store).fill(g)
    assert qb.tree_attention_workspace(c.view, t, group) == 0
    q = torch.randn(b, t, group, dim, generator=g, device="cuda").to(torch.bfloat16)
    rng = np.random.RandomState(8)
    lens = np.where(rng.rand(b) < 0.2, rng.randint(0, cap - 1, b), rng.randint(-1, 3, b))
    lens[0] = cap - t
    _check_attention(qb, c, q, lens, _tree(rng, b, t, absent=True), 0.125)


def test_attention_workspace_of_the_longest_lines(qb):
    """65,535 sequences of 16 heads over 131,200 positions are 1.08 * 10^9 tiles of 128 keys: a plan below 2^31. Twice as long is not."""
    def view(cap, store):
        scale = 1 << 20 if store == "e4m3" else None
        return qb.KVCache(1 << 20, 1 << 20, scale, scale, 16 * cap * 128, cap * 128, _types(qb)[store][0], 65535, 16, 128, cap)

    assert qb.tree_attention_workspace(view(131200, "e4m3"), 1, 16) > 0
    for cap, store in ((262400, "e4m3"), (131200, "bf16")):
        with pytest.raises(qb.QwenError) as e:
            qb.tree_attention_workspace(view(cap, store), 1, 16)
        assert e.value.code == -6


def test_attention_beyond_32_bit_offsets(qb):
    """A cache whose last heads lie more than 2^32 elements from its start."""
    import torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    cap, dim = 1 << 20, 128
    c = Cache(qb, 1, 34, cap, dim, "e4m3")
    g = torch.Generator(device="cuda").manual_seed(2)
    h, length = 33, cap - 5
    assert h * cap * dim > 1 << 32
    part = Cache(qb, 1, 1, cap, dim, "e4m3").fill(g)
    c.k[:, :1], c.v[:, :1], c.ks[:, :1], c.vs[:, :1] = part.k, part.v, part.ks, part.vs
    c.k_all.view(torch.uint8)[:, 1:] = 0
    c.v_all.view(torch.uint8)[:, 1:] = 0
    c.ks[:, 1:], c.vs[:, 1:] = 1.0, 1.0
    c.k.view(torch.uint8)[:, h], c.v.view(torch.uint8)[:, h] = part.k.view(torch.uint8)[:, 0], part.v.view(torch.uint8)[:, 0]
    c.ks[:, h], c.vs[:, h] = part.ks[:, 0], part.vs[:, 0]
    q = torch.randn(1, 2, 34, dim, generator=g, device="cuda").to(torch.bfloat16)
    q[:, :, h] = q[:, :, 0]
    got = _attend(qb, c, q, [length], np.array([[-1, 0]]), 0.1)
    want, tol = _attention64(part, q[:, :, :1].contiguous(), [length], np.array([[-1, 0]]), 0.1)
    assert bool(((got[:, :, :1].double() - want).abs() <= tol).all())
    assert bool(((got[:, :, h:].double() - want).abs() <= tol).all())
    x = torch.randn(1, 3, 34 * dim, generator=g, device="cuda").to(torch.bfloat16)      # rows at the far end
    start = _dev(np.array([cap - 3], np.int32))
    qb.kv_append(c.view, x.data_ptr(), x.data_ptr(), qb.BF16, 34 * dim, 3, start.data_ptr(), 0, _stream())
    back = torch.empty(1, 3, 34 * dim, device="cuda")
    rest = torch.empty_like(back)
    qb.kv_read(c.view, back.data_ptr(), rest.data_ptr(), qb.FP32, 34 * dim, 3, start.data_ptr(), 0, _stream())
    want, a = _codes64(x.double().view(3, 34, dim), "e4m3")
    assert torch.equal(back.view(3, 34, dim), want.float() * a.float())


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def _verify64(logits, draft, tokens, parents, u, temp):
    """The documented walk of one sequence on 64-bit numbers."""
    n, vocab = logits.shape
    path, at = [0], 0
    if parents[0] != -1:
        return [], -1
    while True:
        x = logits[at].astype(np.float64)
        if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf:
            return path, -1
        if temp == 0:
            p = np.zeros(vocab)
            p[int(np.argmax(x))] = 1.0
        else:
            p = np.exp((x - x.max()) / temp)
            p /= p.sum()
        rest, kept = p.copy(), -1
        for i in range(at + 1, n):
            if parents[i] != at or not 0 <= tokens[i] < vocab:
                continue
            t, left = tokens[i], rest.sum()
            q = 1.0 if draft is None or temp == 0 else float(draft[at, t])
            if (0.0 if temp == 0 else float(u[i])) * left * q < rest[t]:
                kept = i
                break
            if draft is None or temp == 0:
                rest[t] = 0.0
            else:
                rest = np.maximum(rest - left * draft[at].astype(np.float64), 0.0)
        if kept < 0:
            w = rest if rest.sum() > 0 else p
            if temp == 0:
                return path, int(np.argmax(p))
            sums = np.cumsum(w)
            over = np.flatnonzero(sums > float(u[0]) * sums[-1])
            return path, int(over[0]) if len(over) else int(np.flatnonzero(w)[-1])
        path.append(kept)
        at = kept


def _verify(qb, logits, draft, tokens, parents, u, temp, pad=0, stream=None):
    """(path, n_path, next) of device tensors logits [b][t][v] and draft; rows `pad` elements further apart than they are long."""
    import torch
    b, t, vocab = logits.shape
    kind = {torch.float32: qb.FP32, torch.bfloat16: qb.BF16, torch.float16: qb.FP16}[logits.dtype]
    lg = torch.full((b, t, vocab + pad), float("nan"), dtype=logits.dtype, device="cuda")
    lg[..., :vocab] = logits
    dr = None
    if draft is not None:
        dr = torch.full((b, t, vocab + pad), float("nan"), device="cuda")
        dr[..., :vocab] = draft
    tk, pr, un = _dev(np.asarray(tokens, np.int32)), _dev(np.asarray(parents, np.int32)), _dev(np.asarray(u, np.float32))
    path = torch.full((b, t), 77, dtype=torch.int32, device="cuda")
    n_path, nxt = torch.full((b,), 77, dtype=torch.int32, device="cuda"), torch.full((b,), 77, dtype=torch.int32, device="cuda")
    qb.tree_verify(lg.data_ptr(), kind, vocab + pad, 0 if dr is None else dr.data_ptr(), vocab + pad, tk.data_ptr(), pr.data_ptr(), un.data_ptr(),
                   b, t, vocab, temp, path.data_ptr(), n_path.data_ptr(), nxt.data_ptr(), _stream() if stream is None else stream)
    torch.cuda.synchronize()
    return path.cpu().numpy(), n_path.cpu().numpy(), nxt.cpu().numpy()


def _check_verify(qb, logits, draft, tokens, parents, u, temp, pad=0):
    got = _verify(qb, logits, draft, tokens, parents, u, temp, pad)
    lg = logits.float().cpu().numpy()
    dr = None if draft is None else draft.cpu().numpy()
    for r in range(lg.shape[0]):
        path, nxt = _verify64(lg[r], None if dr is None else dr[r], tokens[r], parents[r], u[r], temp)
        assert got[0][r].tolist() == path + [-1] * (lg.shape[1] - len(path)), r
        assert (got[1][r], got[2][r]) == (len(path), nxt), r
    return got


def _drafted(seed, b, t, vocab, dtype, with_draft, temp, spread=4.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed)
    logits = (torch.randn(b, t, vocab, generator=g, device="cuda") * spread).to(dtype)
    blurred = logits.float() + 0.5 * torch.randn(logits.shape, generator=g, device="cuda")
    draft = torch.softmax(blurred / (temp or 1.0), -1) if with_draft else None
    par = _tree(rng, b, t)
    par[par < 0] = np.where(rng.rand(int((par < 0).sum())) < 0.3, -2, -1)
    par[:, 0] = -1
    tokens = np.zeros((b, t), np.int32)
    order = torch.sort(blurred, dim=-1, descending=True, stable=True).indices[..., :t].cpu().numpy()
    picks = torch.multinomial(torch.softmax(blurred / (temp or 1.0), -1).view(b * t, vocab), t, replacement=True, generator=g).view(b, t, t).cpu().numpy()
    for r in range(b):
        for i in range(1, t):
            if par[r, i] >= 0:
                s = int((par[r, 1:i] == par[r, i]).sum())
                tokens[r, i] = picks[r, par[r, i], s] if with_draft else order[r, par[r, i], min(s, vocab - 1)]
    return logits, draft, tokens, par, rng.rand(b, t).astype(np.float32)


@pytest.mark.parametrize("temp", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("b,t,vocab,dtype,pad", [(4, 8, 1000, "fp32", 0), (3, 64, 517, "bf16", 3), (40, 5, 4097, "fp32", 1), (5, 12, 33, "fp16", 0),
                                                 (3, 6, 1, "fp32", 2), (160, 3, 130, "fp32", 0), (2, 7, 151936, "fp32", 0), (5, 4, 151936, "bf16", 0),
                                                 (17, 2, 50257, "fp32", 0), (9, 1, 20000, "fp32", 5)])
def test_verify_walks(qb, temp, with_draft, b, t, vocab, dtype, pad):
    case = _drafted(b * 100 + t, b, t, vocab, _types(qb)[dtype][1], with_draft, temp)
    got = _check_verify(qb, *case, temp, pad)
    if t >= 5 and vocab >= 1000 and (temp > 0 or not with_draft):   # (sampled drafts are seldom the greedy token)
        assert got[1].max() > 1      # the cases do keep drafted tokens


@pytest.mark.parametrize("b,dtype,pad", [(150, "fp32", 0), (75, "fp32", 1), (37, "fp32", 0), (20, "bf16", 0)])
def test_verify_rows_beyond_shared_memory(qb, b, dtype, pad):
    """So many sequences that a warp's part of a row no longer fits beside another's, or at all."""
    case = _drafted(b, b, 3, 151936, _types(qb)[dtype][1], b % 2 == 0, 0.7)
    got = _check_verify(qb, *case, 0.7, pad)
    assert got[1].max() > 1


@pytest.mark.parametrize("with_draft", [False, True])
def test_verify_edges_of_the_uniforms(qb, with_draft):
    """Uniforms of 0 and of the largest number below 1; tokens with no probability; masked vocabularies; repeated siblings."""
    import torch
    for seed, u0 in ((1, 0.0), (2, 1.0 - 2.0 ** -24), (3, 0.5)):
        logits, draft, tokens, par, u = _drafted(seed, 6, 9, 700, torch.float32, with_draft, 0.8)
        keep = torch.rand(700, generator=torch.Generator().manual_seed(seed)) < 0.1
        logits[2:, :, ~keep.cuda()] = float("-inf")                # cut by top-k
        if with_draft:
            draft[2:, :, ~keep.cuda()] = 0
            draft = draft / draft.sum(-1, keepdim=True)
        par[3, 1:] = 0                                             # siblings of one root ...
        tokens[3, 1:5] = tokens[3, 1]                              # ... some of them the same token
        tokens[4, 3], tokens[4, 4] = -1, 700                       # no tokens
        u[:, 0] = u0
        u[5] = u0
        _check_verify(qb, logits, draft, tokens, par, u, 0.8)


@pytest.mark.parametrize("vocab,dtype", [(151936, "fp32"), (151936, "bf16"), (1000, "fp32")])
@pytest.mark.parametrize("top", [0.8, 0.95, 0.999, 0.99999])
def test_verify_after_a_likely_token_is_refused(qb, vocab, dtype, top):
    """Chosen drafts: a refused token that had nearly all of the weight leaves little, and the next children are compared with
    exactly that: uniforms at either side of each border decide as in 64 bits."""
    import torch
    b = 48
    g = torch.Generator(device="cuda").manual_seed(vocab + int(top * 1e5))
    logits = torch.randn(b, 5, vocab, generator=g, device="cuda")
    rest = logits[:, 0, 4:].double().exp().sum(-1)
    for i, share in enumerate((0.3, 0.25, 0.2)):                   # of what is left behind token 0
        logits[:, 0, 1 + i] = (rest * share / 0.25).log().float()
    logits[:, 0, 0] = (logits[:, 0, 1:].double().exp().sum(-1) * top / (1 - top)).log().float()
    logits = logits.to(_types(qb)[dtype][1])
    p = torch.softmax(logits[:, 0].double(), -1).cpu().numpy()
    par = np.tile(np.array([-1, 0, 0, 0, 0], np.int32), (b, 1))
    tokens = np.tile(np.array([0, 0, 1, 2, 3], np.int32), (b, 1))
    u = np.random.RandomState(5).rand(b, 5)
    # fp32 sums of the row are off by about 2^-21; what is left behind the first child by 2^-17 at most, or it is summed in 64 bits
    edge = 1e-5
    for r in range(b):
        left = 1 - p[r, 0]
        u[r, 1] = p[r, 0] + 0.5 * left                             # refused
        u[r, 2] = p[r, 1] / left * (1 + (edge if r & 1 else -edge))
        left -= p[r, 1]
        u[r, 3] = p[r, 2] / left * (1 + (edge if r & 2 else -edge))
        left -= p[r, 2]
        u[r, 4] = p[r, 3] / left * (1 + (edge if r & 4 else -edge))
    got = _check_verify(qb, logits, None, tokens, par, u.astype(np.float32), 1.0)
    want = [2 if not r & 1 else 3 if not r & 2 else 4 if not r & 4 else -1 for r in range(b)]
    assert got[0][:, 1].tolist() == want


@pytest.mark.parametrize("temp", [0.0, 1.0])
def test_verify_rows_without_a_distribution(qb, temp):
    import torch
    logits, _, tokens, par, u = _drafted(5, 7, 4, 300, torch.float32, False, temp)
    par[:] = np.array([-1, 0, 1, 2])
    logits[0, 0, 7] = float("nan")
    logits[1, 0, 9] = float("inf")
    logits[2, 0] = float("-inf")
    tokens[3:, 1] = logits[3:, 0].argmax(-1).cpu().numpy()
    u[3:, 1] = 0
    logits[3, 1, 299] = float("nan")                               # reached, and without a distribution
    par[4, 0] = -2                                                 # node 0 is not a root
    par[5, 0] = 0
    got = _check_verify(qb, logits, None, tokens, par, u, temp)
    assert got[2].tolist()[:6] == [-1] * 6 and got[1].tolist()[:6] == [1, 1, 1, 2, 0, 0]


def test_verify_greedy_ties(qb):
    """Equal largest logits: the smaller token, across lanes, warps and CTAs."""
    import torch
    for vocab in (5, 700, 151936):
        logits = torch.zeros(3, 2, vocab, device="cuda")
        logits[1, 0, vocab // 2] = logits[1, 0, vocab - 1] = 2.0
        logits[2] = -1e30
        tokens = np.array([[0, 0], [0, vocab // 2], [0, 1]], np.int32)
        par = np.array([[-1, 0]] * 3, np.int32)
        got = _check_verify(qb, logits, None, tokens, par, np.zeros((3, 2), np.float32), 0.0)
        assert got[2].tolist() == [0, 0, 0] and got[1].tolist() == [2, 2, 1]


def test_verify_draws_follow_the_target(qb):
    """Kept or drawn, the first token after node 0 is distributed as the target's own samples: chi-square over 8 tokens of 20,000
    walks with two drawn children each.  (7 degrees of freedom: a right sampler passes 40 once in a million.)"""
    import torch
    b, n = 20000, 8
    g = torch.Generator(device="cuda").manual_seed(12)
    p = torch.tensor([.3, .2, .15, .12, .1, .06, .05, .02], dtype=torch.float64)
    q = torch.tensor([.05, .3, .05, .2, .1, .1, .1, .1], dtype=torch.float64)
    logits = p.log().float().cuda().expand(b, 3, n).contiguous()
    draft = q.float().cuda().expand(b, 3, n).contiguous()
    tokens = torch.multinomial(draft[:, 0], 3, replacement=True, generator=g).int().cpu().numpy()
    par = np.tile(np.array([-1, 0, 0], np.int32), (b, 1))
    path, n_path, nxt = _verify(qb, logits, draft, tokens, par, np.random.RandomState(3).rand(b, 3).astype(np.float32), 1.0)
    first = np.where(n_path > 1, tokens[np.arange(b), np.maximum(path[:, 1], 0)], nxt)
    seen = np.bincount(first, minlength=n)
    want = p.numpy() * b
    assert (n_path > 1).mean() > 0.5
    assert ((seen - want) ** 2 / want).sum() < 40


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
class _Toy:
    """A one-layer decoder small enough to run in 64 bits: embeddings, q, k, v projections, attention, output logits."""

    def __init__(self, vocab=211, kv=2, group=2, dim=64, seed=0):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda") / math.sqrt(s[0])  # noqa: E731
        self.vocab, self.kv, self.heads, self.dim = vocab, kv, kv * group, dim
        self.e = torch.randn(vocab, 64, generator=g, device="cuda")
        self.wq, self.wk, self.wv = r(64, self.heads * dim) * 2, r(64, kv * dim) * 2, r(64, kv * dim)
        self.wo = r(self.heads * dim, vocab) * 6

    def qkv(self, tokens):
        import torch
        x = self.e[tokens.long()]
        return tuple((x @ w).to(torch.bfloat16) for w in (self.wq, self.wk, self.wv))

    def logits(self, o, tokens):
        return o.float().flatten(-2) @ self.wo + self.e[tokens.long()] @ self.e.T * 0.1


def _greedy_stream(toy, qb, prompt, steps, store):
    """Plain decoding: one token a step through append and attention."""
    import torch
    b, n = prompt.shape
    c = Cache(qb, b, toy.kv, n + steps + 2, toy.dim, store)
    work = torch.empty(qb.tree_attention_workspace(c.view, 1, toy.heads), dtype=torch.uint8, device="cuda")
    root = torch.full((b, 1), -1, dtype=torch.int32, device="cuda")
    q, k, v = toy.qkv(prompt)
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    qb.kv_append(c.view, k.data_ptr(), v.data_ptr(), qb.BF16, toy.kv * toy.dim, n, zero.data_ptr(), 0, _stream())
    out, last = [], prompt[:, -1:].contiguous()
    for i in range(steps):
        at = torch.full((b,), n - 1 + i, dtype=torch.int32, device="cuda")
        q, k, v = toy.qkv(last)
        qb.kv_append(c.view, k.data_ptr(), v.data_ptr(), qb.BF16, toy.kv * toy.dim, 1, at.data_ptr(), 0, _stream())
        o = torch.empty(b, 1, toy.heads, toy.dim, dtype=torch.bfloat16, device="cuda")
        ld = toy.heads * toy.dim
        qb.tree_attention(c.view, q.data_ptr(), o.data_ptr(), qb.BF16, ld, ld, 1, toy.heads, at.data_ptr(), root.data_ptr(), 0.125, work.data_ptr(),
                          work.numel(), _stream())
        last = toy.logits(o, last).argmax(-1).int()
        out.append(last[:, 0].clone())
    return torch.stack(out, 1).cpu().numpy()


@pytest.mark.parametrize("store", ["bf16", "e4m3", "int8"])
def test_drafted_decoding_gives_the_plain_stream(qb, store):
    """A run of all operators: drafted trees (right guesses, wrong guesses, absent nodes) appended, attended, verified and kept, step
    after step, emit the tokens of plain one-token decoding over the same kind of cache."""
    import torch
    toy, b, n, steps, t = _Toy(), 4, 20, 24, 12
    rng = np.random.RandomState(6)
    prompt = _dev(rng.randint(0, toy.vocab, (b, n)).astype(np.int32))
    want = _greedy_stream(toy, qb, prompt, steps + t, store)
    c = Cache(qb, b, toy.kv, n + steps + 2 * t + 2, toy.dim, store)
    work = torch.empty(qb.tree_attention_workspace(c.view, t, toy.heads), dtype=torch.uint8, device="cuda")
    q, k, v = toy.qkv(prompt)
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    qb.kv_append(c.view, k.data_ptr(), v.data_ptr(), qb.BF16, toy.kv * toy.dim, n, zero.data_ptr(), 0, _stream())
    lens = torch.full((b,), n - 1, dtype=torch.int32, device="cuda")
    last, got, kept = prompt[:, -1].cpu().numpy(), [[] for _ in range(b)], 0
    while min(len(x) for x in got) < steps:
        par, tok = np.full((b, t), -2, np.int32), np.zeros((b, t), np.int32)
        for r in range(b):
            par[r, 0], tok[r, 0] = -1, last[r]
            good = 0
            for i in range(1, t - int(rng.randint(0, 3))):
                at = len(got[r]) + int((par[r, :i] == 99).sum())
                if rng.rand() < 0.6 and good >= 0:                 # the right next token below the last right node
                    depth, j = 0, good
                    while j > 0:
                        depth, j = depth + 1, par[r, j]
                    if len(got[r]) + depth < want.shape[1]:
                        par[r, i], tok[r, i], good = good, want[r, len(got[r]) + depth], i
                        continue
                par[r, i], tok[r, i] = rng.randint(0, i), rng.randint(0, toy.vocab)
        tokens, parents = _dev(tok), _dev(par)
        q, k, v = toy.qkv(tokens)
        qb.kv_append(c.view, k.data_ptr(), v.data_ptr(), qb.BF16, toy.kv * toy.dim, t, lens.data_ptr(), 0, _stream())
        o = torch.empty(b, t, toy.heads, toy.dim, dtype=torch.bfloat16, device="cuda")
        ld = toy.heads * toy.dim
        qb.tree_attention(c.view, q.data_ptr(), o.data_ptr(), qb.BF16, ld, ld, t, toy.heads, lens.data_ptr(), parents.data_ptr(), 0.125,
                          work.data_ptr(), work.numel(), _stream())
        logits = toy.logits(o, tokens)
        path = torch.empty(b, t, dtype=torch.int32, device="cuda")
        n_path, nxt = torch.empty(b, dtype=torch.int32, device="cuda"), torch.empty(b, dtype=torch.int32, device="cuda")
        qb.tree_verify(logits.data_ptr(), qb.FP32, toy.vocab, 0, 0, tokens.data_ptr(), parents.data_ptr(), 0, b, t, toy.vocab, 0.0, path.data_ptr(),
                       n_path.data_ptr(), nxt.data_ptr(), _stream())
        qb.kv_keep(c.view, lens.data_ptr(), path.data_ptr(), n_path.data_ptr(), t, _stream())
        lens = lens + n_path
        ph, cnt, last = path.cpu().numpy(), n_path.cpu().numpy(), nxt.cpu().numpy()
        for r in range(b):
            got[r] += [int(tok[r, i]) for i in ph[r, 1:cnt[r]]] + [int(last[r])]
            kept += cnt[r] - 1
    for r in range(b):
        m = min(len(got[r]), steps)
        assert got[r][:m] == want[r, :m].tolist(), r
    assert kept > steps          # drafted tokens were kept


def _step_buffers(qb, store, seed, b=3, t=8, kv=2, group=2, dim=128, vocab=3001, length=150):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"c": Cache(qb, b, kv, length + t, dim, store).fill(g), "b": b, "t": t, "vocab": vocab, "heads": kv * group}
    s["k"], s["v"] = (torch.randn(b, t, kv, dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    s["q"] = torch.randn(b, t, kv * group, dim, generator=g, device="cuda").to(torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    s["lens"] = _dev(np.array([length, 64, 3][:b], np.int32))
    logits, _, tokens, par, u = _drafted(seed, b, t, vocab, torch.float32, False, 1.0)
    s.update(logits=logits, tokens=_dev(tokens), parents=_dev(par), u=_dev(u))
    s["work"] = torch.empty(qb.tree_attention_workspace(s["c"].view, t, s["heads"]), dtype=torch.uint8, device="cuda")
    s["path"] = torch.empty(b, t, dtype=torch.int32, device="cuda")
    s["n_path"], s["next"] = torch.empty(b, dtype=torch.int32, device="cuda"), torch.empty(b, dtype=torch.int32, device="cuda")
    s["back"] = [torch.zeros(b, t, kv, dim, device="cuda") for _ in range(2)]
    return s


def _step(qb, s, stream):
    c, ld = s["c"], s["heads"] * s["c"].dim
    p = lambda n: s[n].data_ptr()  # noqa: E731
    qb.kv_append(c.view, p("k"), p("v"), qb.BF16, c.kv * c.dim, s["t"], p("lens"), 0, stream)
    qb.tree_attention(c.view, p("q"), p("out"), qb.BF16, ld, ld, s["t"], s["heads"], p("lens"), p("parents"), 0.09, p("work"), s["work"].numel(), stream)
    qb.tree_verify(p("logits"), qb.FP32, s["vocab"], 0, 0, p("tokens"), p("parents"), p("u"), s["b"], s["t"], s["vocab"], 1.0, p("path"), p("n_path"),
                   p("next"), stream)
    qb.kv_keep(c.view, p("lens"), p("path"), p("n_path"), s["t"], stream)
    qb.kv_read(c.view, s["back"][0].data_ptr(), s["back"][1].data_ptr(), qb.FP32, c.kv * c.dim, s["t"], p("lens"), p("n_path"), stream)


def _result(s):
    return [x.clone() for x in (s["out"], s["path"], s["n_path"], s["next"], *s["back"])]


@pytest.mark.parametrize("length,t", [(150, 8), (1500, 8), (1500, 40)])
@pytest.mark.parametrize("store", ["bf16", "e4m3"])
def test_captured_step_follows_its_inputs(qb, store, length, t):
    """The step captured into a CUDA graph and replayed on other inputs, lengths and trees equals the eager step bit for bit."""
    import torch
    a, other = _step_buffers(qb, store, 1, t=t, length=length), _step_buffers(qb, store, 2, t=t, length=length)
    _step(qb, a, _stream())                                        # (also: kernels are loaded before the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(qb, a, _stream())
    other["lens"] = _dev(np.array([17, length - 1, 0], np.int32))
    for n in ("k", "v", "q", "lens", "logits", "tokens", "parents", "u"):
        a[n].copy_(other[n])
    for x, y in ((a["c"].k, other["c"].k), (a["c"].v, other["c"].v), (a["c"].ks, other["c"].ks), (a["c"].vs, other["c"].vs)):
        if x is not None:
            x.view(torch.uint8).copy_(y.view(torch.uint8)) if x.dtype.itemsize == 1 else x.copy_(y)
    for x in a["back"]:
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    _step(qb, other, _stream())
    torch.cuda.synchronize()
    for x, y in zip(_result(a), _result(other)):
        assert torch.equal(x, y)
    graph.reset()


@pytest.mark.parametrize("length,t", [(150, 8), (1500, 8), (1500, 40)])
def test_two_streams_and_repeats(qb, length, t):
    """Steps on two streams at once, each with its own workspace, give what they give alone, every time."""
    import torch
    alone = []
    for seed in (3, 4):
        s = _step_buffers(qb, "int8", seed, t=t, length=length)
        _step(qb, s, _stream())
        torch.cuda.synchronize()
        alone.append(_result(s))
    for _ in range(5):
        states, streams = [_step_buffers(qb, "int8", seed, t=t, length=length) for seed in (3, 4)], [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for s, st in zip(states, streams):
            _step(qb, s, st.cuda_stream)
        torch.cuda.synchronize()
        for s, want in zip(states, alone):
            for x, y in zip(_result(s), want):
                assert torch.equal(x, y)


def test_refusals_on_the_device(qb):
    """Host memory, too small a workspace: refused with a message, and the next call works."""
    import torch
    s = _step_buffers(qb, "bf16", 5, length=1500)      # (long enough to need a workspace)
    assert s["work"].numel() > 0
    host = torch.zeros(4096, dtype=torch.int32)
    pinned = torch.zeros(4096, dtype=torch.int32).pin_memory()
    c = s["c"]
    ld = s["heads"] * c.dim
    for bad in (host.data_ptr(), pinned.data_ptr()):
        for f in (lambda: qb.kv_append(c.view, s["k"].data_ptr(), s["v"].data_ptr(), qb.BF16, c.kv * c.dim, s["t"], bad),
                  lambda: qb.kv_keep(c.view, s["lens"].data_ptr(), bad, s["n_path"].data_ptr(), s["t"]),
                  lambda: qb.tree_verify(s["logits"].data_ptr(), qb.FP32, s["vocab"], 0, 0, s["tokens"].data_ptr(), bad, s["u"].data_ptr(), s["b"],
                                         s["t"], s["vocab"], 1.0, s["path"].data_ptr(), s["n_path"].data_ptr(), s["next"].data_ptr())):
            with pytest.raises(qb.QwenError) as e:
                f()
            assert e.value.code == -1 and "device memory" in str(e.value)
    with pytest.raises(qb.QwenError) as e:
        qb.tree_attention(c.view, s["q"].data_ptr(), s["out"].data_ptr(), qb.BF16, ld, ld, s["t"], s["heads"], s["lens"].data_ptr(),
                          s["parents"].data_ptr(), 0.1, s["work"].data_ptr(), s["work"].numel() - 1)
    assert e.value.code == -1 and "workspace" in str(e.value)
    _step(qb, s, _stream())
    torch.cuda.synchronize()
    assert bool(s["out"].isfinite().all())


@pytest.mark.parametrize("b,with_draft,temp,node", [(1, False, 0.0, 0), (1, True, 1.0, 0), (1, False, 1.0, 1), (6, True, 1.0, 1), (37, True, 0.7, 0), (37, True, 0.7, 1)])
def test_verify_reports_a_wait_that_ran_out(qb, b, with_draft, temp, node):
    """A row's copy that never completes: the bounded wait ends, the call returns -1 for the next token of every sequence that waits
    for it, and the next call is right."""
    import torch
    case = _drafted(b, b, 3, 151936, torch.float32, with_draft, temp)
    case[3][:] = np.array([-1, 0, 1])                              # node 1's row is copied while node 0's is read
    qb.debug_draft_wait(5_000_000, node)
    try:
        path, n_path, nxt = _verify(qb, *case, temp)
    finally:
        qb.debug_draft_wait()
    if node == 0:
        assert (nxt == -1).all() and (n_path == 1).all() and (path[:, 0] == 0).all() and (path[:, 1:] == -1).all()
    else:                                                          # those that reached node 1 have no token; the others did not need its row
        want = _check_verify(qb, *case, temp)
        reached = want[1] > 1
        assert (nxt[reached] == -1).all() and (n_path[reached] == 2).all()
        assert ((nxt == want[2]) | (nxt == -1)).all()
    _check_verify(qb, *case, temp)


@pytest.mark.parametrize("store", ["bf16", "e4m3"])
@pytest.mark.parametrize("cap", [200, 1500])
def test_attention_reports_a_wait_that_ran_out(qb, store, cap):
    """K and V that are never announced: the bounded waits end, the call's rows are NaN, and the next call is right."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    t = 40
    c = Cache(qb, 2, 2, cap, 128, store).fill(g)
    q = torch.randn(2, t, 2, 128, generator=g, device="cuda").to(torch.bfloat16)
    par, lens = _tree(np.random.RandomState(1), 2, t), [cap - t, 3]
    qb.debug_draft_wait(5_000_000, 0)
    try:
        got = _attend(qb, c, q, lens, par, 0.1)
    finally:
        qb.debug_draft_wait()
    assert bool(got.isnan().all())
    _check_attention(qb, c, q, lens, par, 0.1)


def test_batch_cache_views_the_slots(qb, checkpoint):
    """qwen_batch_cache: the K/V that the batched prompt pass wrote, read through the view, match between the one-layer and the
    all-layers view, and attention over a slot's layer runs on them."""
    import torch
    e = qb.Engine(checkpoint, 0)
    try:
        with pytest.raises(qb.QwenError) as err:
            e.batch_cache(0)
        assert err.value.code == -7
        e.batch_init(2)
        tokens = np.random.RandomState(0).randint(0, qb.VOCAB_SIZE, 90)
        e.batch_prefill(0, tokens)
        e.batch_prefill(1, tokens[:70])
        for bad in (-2, 28):
            with pytest.raises(qb.QwenError):
                e.batch_cache(bad)
        whole, one = e.batch_cache(), e.batch_cache(5)
        assert (whole.n_kv_heads, one.n_kv_heads, one.capacity, one.n_seqs) == (224, 8, qb.SEQ_LEN, 2)
        zero = torch.zeros(2, dtype=torch.int32, device="cuda")
        a = [torch.zeros(2, 90, 224, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        b = [torch.zeros(2, 90, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        qb.kv_read(whole, a[0].data_ptr(), a[1].data_ptr(), qb.BF16, 224 * 128, 90, zero.data_ptr(), 0, _stream())
        qb.kv_read(one, b[0].data_ptr(), b[1].data_ptr(), qb.BF16, 8 * 128, 90, zero.data_ptr(), 0, _stream())
        for x, y in zip(a, b):
            assert torch.equal(x[:, :, 40:48], y)
            assert bool((y[0].float().abs().amax((1, 2)) > 0).all()) and bool((y[1, 70:] == 0).all())
        q = torch.randn(2, 1, 16, 128, device="cuda").to(torch.bfloat16)
        out = torch.empty_like(q)
        work = torch.empty(qb.tree_attention_workspace(one, 1, 16), dtype=torch.uint8, device="cuda")
        lens, par = _dev(np.array([89, 69], np.int32)), _dev(np.array([[-1], [-1]], np.int32))
        qb.tree_attention(one, q.data_ptr(), out.data_ptr(), qb.BF16, 2048, 2048, 1, 16, lens.data_ptr(), par.data_ptr(), 128 ** -0.5, work.data_ptr(),
                          work.numel(), _stream())
        for r, n in ((0, 90), (1, 70)):
            k, v = (x[r, :n].double().transpose(0, 1).repeat_interleave(2, 0) for x in b)
            w = torch.softmax(torch.einsum("hd,hkd->hk", q[r, 0].double(), k) * 128 ** -0.5, -1)
            want = torch.einsum("hk,hkd->hd", w, v)
            mag = torch.einsum("hk,hkd->hd", w, v.abs())
            # the output's and the weights' bf16 roundings (2^-8 each), and 2^-12 for the fp32 scores of these sizes
            assert bool(((out[r, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mag).all())
    finally:
        e.close()
