"""Refusals of the operators of serving over pages that need no GPU: every bad size, type,
stride, NULL and misaligned pointer is turned down with a status and a message before the
device is touched."""
import ctypes

import pytest

OK_PTR = 1 << 20    # 16-byte aligned, never followed: the calls below end before


def _view(qb, **over):
    f = dict(k=OK_PTR, v=OK_PTR, k_scale=None, v_scale=None, table=OK_PTR, page_stride=2 * 16 * 128, head_stride=16 * 128, dtype=qb.BF16, n_pages=10, n_seqs=3,
             n_kv_heads=2, head_dim=128, page_size=16, max_pages=8)
    f.update(over)
    return qb.KVPages(*[f[n] for n, _ in qb.KVPages._fields_])


def _raises(qb, code, f, *a):
    with pytest.raises(qb.QwenError) as e:
        f(*a)
    assert e.value.code == code, str(e.value)
    assert len(str(e.value)) > 15


ROPE = dict(q=OK_PTR, k=OK_PTR, v=OK_PTR, dtype=0, ldq=512, ldk=256, ldv=256, n_rows=5, n_heads=4, n_kv_heads=2, head_dim=128, q_gain=OK_PTR, k_gain=OK_PTR, gain_dtype=0,
            eps=1e-6, base=1e6, positions=OK_PTR, q_out=OK_PTR, k_out=OK_PTR, out_dtype=0, ldqo=512, ldko=256)
PAGED = dict(q=OK_PTR, out=OK_PTR + 16, dtype=0, ldq=512, ldo=512, n_heads=4, lens=OK_PTR, scale=0.1, work=OK_PTR, work_bytes=1 << 30)


@pytest.mark.parametrize("over,code", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(k=OK_PTR + 8), -1), (dict(v=OK_PTR + 2), -1), (dict(table=None), -1), (dict(table=OK_PTR + 2), -1), (dict(dtype=2), -1),
    (dict(dtype=9), -1), (dict(dtype=-1), -1), (dict(head_dim=96), -6), (dict(head_dim=0), -6), (dict(n_seqs=0), -1), (dict(n_seqs=65536), -1), (dict(n_kv_heads=0), -1),
    (dict(n_pages=0), -1), (dict(page_size=0), -1), (dict(page_size=24), -1), (dict(page_size=1 << 17), -1), (dict(max_pages=0), -1), (dict(max_pages=1 << 27), -1),
    (dict(head_stride=15 * 128), -1), (dict(page_stride=15 * 128), -1), (dict(head_stride=16 * 128 + 8), -1), (dict(page_stride=-4096), -1), (dict(k_scale=OK_PTR), -1),
    (dict(dtype=3), -1), (dict(dtype=4, k_scale=OK_PTR), -1), (dict(dtype=3, k_scale=OK_PTR + 2, v_scale=OK_PTR), -1)])
def test_bad_views(qb, over, code):
    _raises(qb, code, qb.qk_rope, *ROPE.values(), _view(qb, **over), OK_PTR)
    _raises(qb, code, qb.paged_attention, _view(qb, **over), *PAGED.values())
    if not set(over) & {"k", "v", "table", "k_scale"} and over != dict(dtype=3):
        _raises(qb, code, qb.paged_attention_workspace, _view(qb, **over), 4)


@pytest.mark.parametrize("over,code", [
    (dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1), (dict(q=OK_PTR + 8), -1), (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(out_dtype=4), -1), (dict(ldq=504), -1),
    (dict(ldq=513), -1), (dict(ldk=255), -1), (dict(ldv=128), -1), (dict(ldqo=256), -1), (dict(ldko=252), -1), (dict(n_rows=0), -1), (dict(n_rows=-3), -1), (dict(n_heads=0), -1),
    (dict(n_heads=5), -1), (dict(n_kv_heads=0), -1), (dict(head_dim=96), -6), (dict(q_gain=0), -1), (dict(k_gain=0), -1), (dict(gain_dtype=3), -1), (dict(k_gain=OK_PTR + 2), -1),
    (dict(eps=-1e-6), -1), (dict(eps=float("nan")), -1), (dict(eps=float("inf")), -1), (dict(base=0.5), -1), (dict(base=float("nan")), -1), (dict(base=float("inf")), -1),
    (dict(positions=0), -1), (dict(q_out=0), -1), (dict(q_out=OK_PTR + 4), -1), (dict(k_out=OK_PTR + 4), -1), (dict(ldq=(1 << 36) + 8), -1)])
def test_bad_rope(qb, over, code):
    _raises(qb, code, qb.qk_rope, *{**ROPE, **over}.values(), _view(qb), OK_PTR)


@pytest.mark.parametrize("out,other,paged", [("q_out", "q", True), ("q_out", "k", True), ("q_out", "v", True), ("k_out", "q", True), ("k_out", "k", True), ("k_out", "v", True),
                                             ("q_out", "k_out", True), ("q_out", "q", False), ("k_out", "k", False), ("q_out", "k_out", False)])
def test_rope_outputs_apart(qb, out, other, paged):
    """Outputs in the place of an input, or of each other; apart, the call gets as far as the device."""
    apart = {**ROPE, **{n: OK_PTR + (i << 20) for i, n in enumerate(("q", "k", "v", "q_out", "k_out"))}}
    pages = (_view(qb), OK_PTR) if paged else ()
    with pytest.raises(qb.QwenError) as e:
        qb.qk_rope(*{**apart, out: apart[other]}.values(), *pages)
    assert e.value.code == -1 and "must not be" in str(e.value)
    with pytest.raises(qb.QwenError) as e:
        qb.qk_rope(*apart.values(), *pages)
    assert "must not be" not in str(e.value)


def test_bad_rope_pages(qb):
    _raises(qb, -1, qb.qk_rope, *ROPE.values(), _view(qb), 0)
    _raises(qb, -1, qb.qk_rope, *ROPE.values(), _view(qb, n_kv_heads=1), OK_PTR)
    _raises(qb, -1, qb.qk_rope, *ROPE.values(), _view(qb, head_dim=64), OK_PTR)


PROMPT = dict(q=OK_PTR, k=OK_PTR, v=OK_PTR, out=OK_PTR + 16, dtype=0, ldq=512, ldk=256, ldv=256, ldo=512, starts=OK_PTR, k_starts=0, n_seqs=2, n_rows=10, n_keys=10, n_heads=4,
              n_kv_heads=2, head_dim=128, scale=0.1)


@pytest.mark.parametrize("over,code", [
    (dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1), (dict(out=0), -1), (dict(out=OK_PTR), -1), (dict(q=OK_PTR + 8), -1), (dict(k=OK_PTR + 2), -1), (dict(dtype=2), -1),
    (dict(dtype=3), -1), (dict(ldq=504), -1), (dict(ldk=250), -1), (dict(ldv=8), -1), (dict(ldo=515), -1), (dict(starts=0), -1), (dict(starts=OK_PTR + 2), -1),
    (dict(k_starts=OK_PTR + 1), -1), (dict(n_seqs=0), -1), (dict(n_seqs=65536), -1), (dict(n_rows=0), -1), (dict(n_keys=0), -1), (dict(n_heads=3), -1), (dict(n_heads=0), -1),
    (dict(n_heads=258, ldq=129 * 256, ldo=129 * 256), -6), (dict(head_dim=32), -6), (dict(scale=float("nan")), -1), (dict(scale=2.0 ** 127), -1), (dict(n_rows=(1 << 30) + 1), -1)])
def test_bad_prompt(qb, over, code):
    _raises(qb, code, qb.prompt_attention, *{**PROMPT, **over}.values())


@pytest.mark.parametrize("over,code", [
    (dict(q=0), -1), (dict(q=OK_PTR + 8), -1), (dict(out=0), -1), (dict(out=OK_PTR), -1), (dict(dtype=1), -1), (dict(dtype=2), -1), (dict(ldq=504), -1), (dict(ldo=511), -1),
    (dict(n_heads=0), -1), (dict(n_heads=3), -1), (dict(n_heads=2 << 15, ldq=1 << 24, ldo=1 << 24), -6), (dict(lens=0), -1), (dict(lens=OK_PTR + 2), -1), (dict(scale=float("inf")), -1),
    (dict(work=OK_PTR + 4), -1)])
def test_bad_paged(qb, over, code):
    _raises(qb, code, qb.paged_attention, _view(qb), *{**PAGED, **over}.values())


def test_short_tables_need_no_workspace(qb):
    assert qb.paged_attention_workspace(_view(qb), 4) == 0
    assert qb.load_library().qwen_paged_attention_workspace(ctypes.byref(_view(qb)), 4, None) == -1


SCORE = dict(logits=OK_PTR, dtype=2, ld=100, n_rows=3, vocab=100, tokens=OK_PTR, temperature=1.0, n_top=4, logprob=OK_PTR, entropy=OK_PTR, top_ids=OK_PTR, top_logprobs=OK_PTR)


@pytest.mark.parametrize("over", [
    dict(logits=0), dict(logits=OK_PTR + 2), dict(dtype=3), dict(ld=99), dict(n_rows=0), dict(vocab=0), dict(tokens=0), dict(logprob=0), dict(tokens=OK_PTR + 1), dict(temperature=0.0),
    dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1e7), dict(n_top=-1), dict(n_top=65), dict(top_ids=0), dict(top_logprobs=0), dict(entropy=OK_PTR + 2),
    dict(tokens=0, logprob=0, entropy=0, n_top=0), dict(n_rows=(1 << 24) + 1)])
def test_bad_logprobs(qb, over):
    _raises(qb, -1, qb.token_logprobs, *{**SCORE, **over}.values())
