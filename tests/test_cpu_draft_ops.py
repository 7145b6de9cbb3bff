"""Refusals of the drafted-token operators that need no GPU: every bad size, type,
stride, NULL and misaligned pointer is turned down with a status and a message
before the device is touched."""
import ctypes
import os
import re
from decimal import Decimal, getcontext

import pytest

from conftest import PKG

OK_PTR = 1 << 20    # 16-byte aligned, never followed: the calls below end before


def _view(qb, **over):
    f = dict(k=OK_PTR, v=OK_PTR, k_scale=None, v_scale=None, seq_stride=64 * 128 * 2, head_stride=64 * 128, dtype=qb.BF16, n_seqs=3,
             n_kv_heads=2, head_dim=128, capacity=64)
    f.update(over)
    return qb.KVCache(*[f[n] for n, _ in qb.KVCache._fields_])


BAD_VIEWS = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(k=OK_PTR + 8), -1), (dict(v=OK_PTR + 2), -1), (dict(dtype=2), -1), (dict(dtype=9), -1),
    (dict(dtype=-1), -1), (dict(head_dim=96), -6), (dict(head_dim=0), -6), (dict(n_seqs=0), -1), (dict(n_seqs=65536), -1),
    (dict(n_kv_heads=0), -1), (dict(capacity=0), -1), (dict(head_stride=64 * 128 - 128), -1), (dict(seq_stride=64 * 128 - 128), -1),
    (dict(head_stride=64 * 128 + 8), -1), (dict(seq_stride=-64 * 128), -1), (dict(k_scale=OK_PTR), -1), (dict(dtype=3), -1),
    (dict(dtype=4, k_scale=OK_PTR), -1), (dict(dtype=3, k_scale=OK_PTR + 2, v_scale=OK_PTR), -1),
]


def _raises(qb, code, f, *a):
    with pytest.raises(qb.QwenError) as e:
        f(*a)
    assert e.value.code == code, str(e.value)
    assert len(str(e.value)) > 15


@pytest.mark.parametrize("over,code", BAD_VIEWS)
def test_bad_views(qb, over, code):
    c = _view(qb, **over)
    _raises(qb, code, qb.kv_append, c, OK_PTR, OK_PTR, qb.BF16, 256, 4, OK_PTR)
    _raises(qb, code, qb.kv_read, c, OK_PTR, OK_PTR, qb.BF16, 256, 4, OK_PTR)
    _raises(qb, code, qb.kv_keep, c, OK_PTR, OK_PTR, OK_PTR, 4)
    _raises(qb, code, qb.tree_attention, c, OK_PTR, OK_PTR + 16, qb.BF16, 512, 512, 4, 4, OK_PTR, OK_PTR, 0.1, OK_PTR, 1 << 30)


@pytest.mark.parametrize("args", [
    (0, OK_PTR, 0, 256, 4, OK_PTR), (OK_PTR, 0, 0, 256, 4, OK_PTR), (OK_PTR + 4, OK_PTR, 0, 256, 4, OK_PTR), (OK_PTR, OK_PTR, 3, 256, 4, OK_PTR),
    (OK_PTR, OK_PTR, 0, 248, 4, OK_PTR), (OK_PTR, OK_PTR, 0, 257, 4, OK_PTR), (OK_PTR, OK_PTR, 0, 256, 0, OK_PTR),
    (OK_PTR, OK_PTR, 0, 256, 65, OK_PTR), (OK_PTR, OK_PTR, 0, 256, 4, 0), (OK_PTR, OK_PTR, 0, 256, 4, OK_PTR + 2),
    (OK_PTR, OK_PTR, 0, 256, 4, OK_PTR, OK_PTR + 1)])
def test_bad_rows(qb, args):
    _raises(qb, -1, qb.kv_append, _view(qb), *args)
    _raises(qb, -1, qb.kv_read, _view(qb), *args)


@pytest.mark.parametrize("args", [(0, OK_PTR, OK_PTR, 4), (OK_PTR, 0, OK_PTR, 4), (OK_PTR, OK_PTR, 0, 4), (OK_PTR, OK_PTR, OK_PTR, 0),
                                  (OK_PTR, OK_PTR, OK_PTR, 65)])
def test_bad_keep(qb, args):
    _raises(qb, -1, qb.kv_keep, _view(qb), *args)


GOOD = dict(q=OK_PTR, out=OK_PTR + 16, dtype=0, ldq=512, ldo=512, n_nodes=4, n_heads=4, lens=OK_PTR, parents=OK_PTR, scale=0.1, work=OK_PTR,
            work_bytes=1 << 30)


@pytest.mark.parametrize("over", [
    dict(q=0), dict(q=OK_PTR + 8), dict(out=0), dict(out=OK_PTR), dict(dtype=1), dict(dtype=2), dict(ldq=504), dict(ldq=513), dict(ldo=511),
    dict(n_nodes=0), dict(n_nodes=65), dict(n_heads=0), dict(n_heads=3), dict(lens=0), dict(parents=OK_PTR + 1), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(work=0), dict(work=OK_PTR + 4)])
def test_bad_attention(qb, over):
    big = _view(qb, capacity=4096, head_stride=4096 * 128, seq_stride=2 * 4096 * 128)
    _raises(qb, -1, qb.tree_attention, big, *{**GOOD, **over}.values())


@pytest.mark.parametrize("scale", [2.0 ** 127, -2.4e38, 3.4e38])
def test_attention_scales_whose_base_2_form_overflows(qb, scale):
    big = _view(qb, capacity=4096, head_stride=4096 * 128, seq_stride=2 * 4096 * 128)
    _raises(qb, -1, qb.tree_attention, big, *{**GOOD, "scale": scale, "parents": 0}.values())
    with pytest.raises(qb.QwenError, match="scale"):
        qb.tree_attention(big, *{**GOOD, "scale": scale, "parents": 0}.values())


def test_small_caches_need_no_workspace(qb):
    assert qb.tree_attention_workspace(_view(qb), 4, 4) == 0
    _raises(qb, -1, qb.tree_attention, _view(qb), *{**GOOD, "work": OK_PTR + 4}.values())


def test_bad_workspace_queries(qb):
    for c, t, h in ((_view(qb), 0, 4), (_view(qb), 65, 4), (_view(qb), 4, 5), (_view(qb, n_seqs=0), 4, 4)):
        _raises(qb, -1, qb.tree_attention_workspace, c, t, h)
    assert qb.load_library().qwen_tree_attention_workspace(ctypes.byref(_view(qb)), 4, 4, None) == -1


VERIFY = dict(logits=OK_PTR, dtype=2, ld=100, draft=0, ld_draft=0, tokens=OK_PTR, parents=OK_PTR, u=OK_PTR, n_seqs=2, n_nodes=4, vocab=100,
              temperature=1.0, path=OK_PTR, n_path=OK_PTR, next=OK_PTR)


@pytest.mark.parametrize("over", [
    dict(logits=0), dict(logits=OK_PTR + 2), dict(dtype=3), dict(ld=99), dict(draft=OK_PTR, ld_draft=99), dict(draft=OK_PTR + 1, ld_draft=100),
    dict(tokens=0), dict(parents=0), dict(u=0), dict(n_seqs=0), dict(n_seqs=65536), dict(n_nodes=0), dict(n_nodes=65), dict(vocab=0),
    dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1e-9), dict(temperature=float("inf")), dict(path=0),
    dict(n_path=OK_PTR + 2), dict(next=0)])
def test_bad_verify(qb, over):
    _raises(qb, -1, qb.tree_verify, *{**VERIFY, **over}.values())


def test_batch_cache_needs_a_handle(qb):
    assert qb.load_library().qwen_batch_cache(None, 0, ctypes.byref(qb.KVCache())) == -1


@pytest.mark.parametrize("args", [(999_999, 0), (1, -1), (0, -2), (0, 64)])
def test_bad_debug_wait(qb, args):
    _raises(qb, -1, qb.debug_draft_wait, *args)
    qb.debug_draft_wait()


def test_power_of_two_polynomial():
    """The verification's fp64 powers of two: its coefficients interpolate 2^f at the nine Chebyshev nodes of [-1/2, 1/2], and are
    within 2^-39 of it."""
    src = open(os.path.join(PKG, "csrc", "tree_verify.cuh")).read()
    low = [float(x) for x in re.search(r"kC\[8\] = \{([^}]*)\}", src).group(1).split(",")]
    c = [float(re.search(r"fma\(f\[j\], ([0-9.e-]+), kC\[0\]\)", src).group(1))] + low      # highest power first
    getcontext().prec = 50
    ln2 = Decimal(2).ln()
    cosines = [Decimal("0.98480775301220805936674302458952"), Decimal("0.86602540378443864676372317075294"),
               Decimal("0.64278760968653932632264340990726"), Decimal("0.34202014332566873304409961468226")]
    nodes = [x / 2 for x in cosines] + [Decimal(0)] + [-x / 2 for x in cosines]                # cos((2 k + 1) 10 degrees) / 2
    table, newton = [(x * ln2).exp() for x in nodes], []
    for i in range(9):                                                                         # divided differences
        newton.append(table[0])
        table = [(table[k + 1] - table[k]) / (nodes[k + 1 + i] - nodes[k]) for k in range(len(table) - 1)]
    want = [newton[8]]
    for i in range(7, -1, -1):                                                                 # (...) (f - node) + difference, expanded
        want = [a - b * nodes[i] for a, b in zip(want + [Decimal(0)], [Decimal(0)] + want)]
        want[-1] += newton[i]
    for a, b in zip(c, want):
        assert abs(Decimal(a) - b) <= Decimal(2) ** -48 * abs(b), (a, b)      # (the stored numbers have 16 or 17 digits of a 64-bit solution)
    worst = 0.0
    for k in range(-500, 501):
        f, y = k / 1000, 0.0
        for a in c:
            y = y * f + a
        worst = max(worst, abs(float(Decimal(y) / (Decimal(k) / 1000 * ln2).exp() - 1)))
    assert worst <= 2.0 ** -39, worst
