"""The generation operators where their numerics or their bookkeeping are at their limits: few bits of the softmax weights,
value scales far apart, keys of very different lengths, long sequences, rows that are cut off, graph capture."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_generation import (EPS16, RefCache, TYPES, _gen, _randn, attention_ref, db, new_cache)  # noqa: E402,F401


def cached_rows(db, dtype, k, v, q, scale=128 ** -0.5, before=0, cache=None):
    """One item: its first `before` tokens appended, then the others with their queries q -> (outputs, the 64-bit reference)."""
    n, Hk = k.shape[:2]
    c = cache or new_cache(db, 1, Hk, dtype, n, _gen(1))
    at = torch.full((1,), before, dtype=torch.int32, device="cuda")
    if before:
        db.kv8_append(c, k[:before], v[:before], torch.zeros_like(at))
    db.kv8_append(c, k[before:], v[before:], at)
    out = db.kv8_attention(c, q, at, scale=scale)
    ref = RefCache(1, Hk, TYPES[dtype])
    ref.append(k, v, [n])
    return out, attention_ref(ref.values(ref.k[0]), ref.values(ref.v[0]), q.cpu(), scale)


def check_rows(out, want, dtype):
    """As check_attention, with each row's and head's own RMS as the floor."""
    err = (out.double().cpu() - want).abs()
    bound = 2 * EPS16[dtype] * (want.abs() + want.square().mean(-1, keepdim=True).sqrt())
    assert torch.all(err <= bound), float((err / bound).max())


@pytest.mark.parametrize("rows,before", [(2, 20), (2, 300), (4, 300), (100, 0), (40, 300)])
def test_cache_weights_keep_their_bits(db, rows, before):
    """bf16 outputs are the 64-bit result rounded once.  A weight's error of d moves an output by d of its terms; a rounding
    then differs where the result lies that close to the middle of two bf16 values, some 2 d / 2^-8 of all outputs.  Scores
    and weights in 32 bits leave d near 2^-18 (scores up to 16, 8 sums of 2^-24 each): one output in 500; one in 100 is
    allowed.  (Weights of 11 bits, d near 2^-13, give one in 20.)"""
    gen, Hk, group = _gen(rows + before), 2, 4
    k, v = (_randn(gen, before + rows, Hk, 128, dtype=torch.bfloat16) for _ in range(2))
    q = _randn(gen, rows, Hk * group, 128, dtype=torch.bfloat16)
    out, want = cached_rows(db, "bf16", k, v, q, before=before)
    check_rows(out, want, "bf16")
    differ = (out.cpu() != want.to(torch.bfloat16)).double().mean().item()
    assert differ <= 0.01, differ
