"""The generation operators where their numerics or their bookkeeping are at their limits: few bits of the softmax weights,
value scales far apart, keys of very different lengths, long sequences, rows that are cut off, graph capture."""
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_generation import (EPS16, RefCache, TYPES, _gen, _randn, attention_ref, check_delta, db,  # noqa: E402
                                 delta_inputs, delta_ref, new_cache, rules_ref)  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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
    """As check_attention, with each row's and head's own RMS as the floor; f16 outputs below 2^-14 lie 2^-24 apart."""
    err = (out.double().cpu() - want).abs()
    bound = 2 * EPS16[dtype] * (want.abs() + want.square().mean(-1, keepdim=True).sqrt()) + (2.0 ** -24 if dtype == "f16" else 0)
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


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 4, 30])
def test_cache_weak_keys_add_up(db, dtype, rows):
    """One key holds nearly all of the softmax and has no value (what models do with their first token): the output is the
    sum of 8000 weights of 2^-24.5 each."""
    gen, Hk, group, n = _gen(21), 1, 4, 8005
    k = torch.zeros(n, Hk, 128, dtype=TYPES[dtype], device="cuda")
    k[0] = 17.0 / 128 ** 0.5
    v = _randn(gen, 1, Hk, 128, dtype=TYPES[dtype], scale=50.0).repeat(n, 1, 1)
    v[0] = 0
    q = torch.ones(rows, Hk * group, 128, dtype=TYPES[dtype], device="cuda")
    out, want = cached_rows(db, dtype, k, v, q, before=n - rows)
    check_rows(out, want, dtype)


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_cache_value_scales_far_apart(db, rows):
    """Blocks of 1e-30, of some units and of 1e20 in one sequence, every row against its own terms."""
    gen, Hk, group, n = _gen(12), 1, 4, 230
    k, v = (_randn(gen, n, Hk, 128, dtype=torch.bfloat16) for _ in range(2))
    v[:64] *= 1e-30
    v[128:192] *= 1e20
    for before in (64 - rows // 2 - 1, 128 - rows // 2 - 1, 180, n - rows):
        q = _randn(gen, rows, Hk * group, 128, dtype=torch.bfloat16)
        out, want = cached_rows(db, "bf16", k[:before + rows], v[:before + rows], q, before=before)
        check_rows(out, want, "bf16")


@pytest.mark.parametrize("dtype,base", [("bf16", 1.0), ("f16", 1.0), ("f16", 2.0 ** 12)])
@pytest.mark.parametrize("power", [-22, -20, -18, -16, -12, -4, 4, 12, 20])
def test_cache_a_later_block_changes_no_earlier_row(db, dtype, base, power):
    """256 rows at once; the second block's values are 2^-power of the others'.  Rows are as accurate as their own keys
    allow, and what comes after a row does not reach it.  (base: the larger values; 2^12 keeps f16 outputs out of its
    subnormals.)"""
    if base > 1 and power > 0:
        pytest.skip("the later block would pass f16's largest value")
    gen, Hk, n = _gen(31 + power), 2, 256
    q, k, v = (_randn(gen, n, Hk, 128, dtype=TYPES[dtype]) for _ in range(3))
    v = (v.float() * base * (2.0 ** power if power < 0 else 1.0)).to(TYPES[dtype])
    v[64:128] = (v[64:128].float() * 2.0 ** -power).to(TYPES[dtype])
    out, want = cached_rows(db, dtype, k, v, q)
    check_rows(out, want, dtype)
    w = v.clone()
    w[128:] = (w[128:].float() * 256).to(TYPES[dtype])
    again, _ = cached_rows(db, dtype, k, w, q)
    assert torch.equal(out[:128], again[:128])


def test_cache_scale_of_zero(db):
    """Codes that another program wrote under a scale of 0 are zeros, beside other blocks and alone."""
    gen, Hk = _gen(41), 1
    q, k, v = (_randn(gen, 128, Hk, 128, dtype=torch.bfloat16) for _ in range(3))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    for rows in (2, 128):
        c = new_cache(db, 1, Hk, "bf16", 128, gen)
        db.kv8_append(c, k, v, zero)
        c.v_scales[c.page_table[0, 0].long()] = 0
        got_k, got_v = (x[0].cpu() for x in db.kv8_read(c, zero + 128, 128))
        out = db.kv8_attention(c, q[-rows:], zero + 128 - rows)
        check_rows(out, attention_ref(got_k, got_v, q[-rows:].cpu(), 128 ** -0.5), "bf16")
        assert rows < 128 or not out[:64].any()

@pytest.mark.parametrize("dtype,values,keys", [("bf16", 6.0, 0.0), ("bf16", 2.0, 3.0), ("f16", 1.5, 1.0)])
@pytest.mark.parametrize("rows,before", [(4, 20), (50, 0), (60, 40)])
def test_cache_open_block_is_exact(db, dtype, values, keys, rows, before):
    """Tokens of the open block whose keys and values differ by many powers of ten: each row has the accuracy of what it sees.
    Weights in 16 bits or more (2^-17, twice for their sum), scores from 8 sums of 2^-23 of their terms, the output's own
    rounding; and weights of the full block end at 2^-30 of the largest (f16's last bit, 2^-25, under 2^5)."""
    gen, Hk, group, n = _gen(91 + rows), 2, 4, before + rows
    k, v = (_randn(gen, n, Hk, 128) for _ in range(2))
    k = (k * torch.exp(keys * _randn(gen, n, 1, 1)).clamp(max=1e3)).to(TYPES[dtype])
    v = (v * torch.exp(values * _randn(gen, n, 1, 1)).clamp(max=1e3 if dtype == "f16" else 1e30)).to(TYPES[dtype])
    q = _randn(gen, rows, Hk * group, 128, dtype=TYPES[dtype], scale=0.3)
    out, want = cached_rows(db, dtype, k, v, q, before=before)
    ref = RefCache(1, Hk, TYPES[dtype])
    ref.append(k, v, [n])
    k64, v64, q64 = ref.values(ref.k[0]).double(), ref.values(ref.v[0]).double(), q.double().cpu()
    for i in range(rows):
        seen = before + i + 1
        for h in range(Hk * group):
            kh, vh = k64[:seen, h // group], v64[:seen, h // group]
            weights = torch.softmax((kh @ q64[i, h]) * 128 ** -0.5, 0)
            terms, size = weights @ vh.abs(), (kh.abs() @ q64[i, h].abs()).max().item() * 128 ** -0.5
            bound = EPS16[dtype] * want[i, h].abs() + (2 * 2.0 ** -17 + 2 * 1.45 * size * 2.0 ** -20) * terms
            bound += vh.abs().sum(0) * 2.0 ** -30 + (2.0 ** -24 if dtype == "f16" else 0)
            err = (out[i, h].double().cpu() - want[i, h]).abs()
            assert torch.all(err <= bound), (i, h, float((err / bound).nan_to_num().max()))


@pytest.mark.parametrize("rows", [2, 40])
def test_cache_open_block_under_a_far_larger_one(db, rows):
    """Values of 1e-12 after a block of 1e20: they may end at 2^-100 of it, but come out no larger than they are."""
    gen, Hk, n = _gen(95), 1, 64 + 45
    k, v = (_randn(gen, n, Hk, 128, dtype=torch.bfloat16) for _ in range(2))
    v[:64] *= 1e20
    v[:64, :, 64:] = 0
    v[64:] *= 1e-12
    q = _randn(gen, rows, Hk * 4, 128, dtype=torch.bfloat16)
    out, want = cached_rows(db, "bf16", k, v, q, before=n - rows)
    check_rows(out[..., :64], want[..., :64], "bf16")
    small, exact = out[..., 64:].double().cpu(), want[..., 64:]
    assert torch.all((small - exact).abs() <= 2 * EPS16["bf16"] * exact.abs() + 1e20 * 2.0 ** -100)
    assert small.abs().max() < 1e-10


@pytest.mark.parametrize("short", [1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("size", [1.0, 8.0])
@pytest.mark.parametrize("T", [64, 130])
def test_delta_one_short_key(db, T, size, short):
    """f16 keys as they come from a projection: one far shorter than the others costs the others nothing."""
    gen, Hk, Hv = _gen(51), 1, 2
    q, k, v, g, beta = delta_inputs(gen, T, Hk, Hv, torch.float16, decay=0.01)
    k = (k.float() * size).half()
    k[20] = (k[20].float() * short).half()
    s = _randn(gen, 1, Hv, 128, 128, scale=0.3)
    got = db.gated_delta(q, k, v, g, beta, state=s)
    check_delta(got, delta_ref(q, k, v, g, beta, [T], s, 128 ** -0.5, 1e-6), "f16")


@pytest.mark.parametrize("dtype,large", [("bf16", 1.0), ("f16", 2.0 ** 12)])
@pytest.mark.parametrize("T", [64, 150])
def test_delta_small_values_before_large_ones(db, T, dtype, large):
    """The first tokens' values are 2^-20 of the later ones', in every feature: their outputs are as accurate as alone."""
    gen, Hk, Hv = _gen(53), 1, 2
    q, k, v, g, beta = delta_inputs(gen, T, Hk, Hv, TYPES[dtype])
    v = (v.float() * large).to(TYPES[dtype])
    v[:40] = (v[:40].float() * 2.0 ** -20).to(TYPES[dtype])
    out, _ = db.gated_delta(q, k, v, g, beta)
    want, _ = delta_ref(q, k, v, g, beta, [T], None, 128 ** -0.5, 1e-6)
    for part in (slice(0, 40), slice(40, T)):
        err, rms = (out[part].double().cpu() - want[part]).abs(), want[part].square().mean().sqrt().item()
        bound = 2 * EPS16[dtype] * (want[part].abs() + rms) + (2.0 ** -24 if dtype == "f16" else 0)
        assert torch.all(err <= bound), float((err / bound).max())


@pytest.mark.parametrize("T", [3, 70])
def test_delta_states_side_by_side(db, T):
    """Initial and final states in one buffer, next to one another or the same, give what separate ones give."""
    gen, Hk, Hv, B = _gen(52), 1, 2, 2
    q, k, v, g, beta = delta_inputs(gen, B * T, Hk, Hv, torch.bfloat16)
    pool = _randn(gen, 5, Hv, 128, 128, scale=0.3)
    for first, last, shared in ((0, 2, False), (2, 0, False), (3, 3, False), (2, 0, True), (1, 2, True), (0, 3, True)):
        mine = pool.clone()
        start = mine[first:first + (1 if shared else B)]
        want_out, want = db.gated_delta(q, k, v, g, beta, items=B, state=start.clone())
        out, got = db.gated_delta(q, k, v, g, beta, items=B, state=start, state_out=mine[last:last + B])
        assert torch.equal(out, want_out) and torch.equal(got, want)


@pytest.mark.parametrize("rows", [3, 40])
def test_cache_rows_cut_off_are_zero(db, rows):
    """Rows past max_rows, past the table, or of an item without room are 0, and the error word says so."""
    gen, Hk, Hq = _gen(61), 1, 4
    n = 2 * rows
    q, k, v = (_randn(gen, n, h, 128, dtype=torch.float16) for h in (Hq, Hk, Hk))
    cu = torch.tensor([0, rows, n], dtype=torch.int32, device="cuda")

    def call(lengths, most, cu):
        c = new_cache(db, 2, Hk, "f16", 64, gen)  # two or three blocks
        lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        assert db.device_error_word() == 0
        db.kv8_append(c, k, v, lengths, cu_seqlens=cu, max_rows=most)
        assert db.device_error_word() == 0x10
        out = db.kv8_attention(c, q, lengths, cu_seqlens=cu, max_rows=most, out=torch.full_like(q, 7.0))
        assert db.device_error_word() == 0x10
        return out, c.table_width * 64

    out, _ = call([0, 0], rows - 1, cu)
    _, want = cached_rows(db, "f16", k[:rows - 1], v[:rows - 1], q[:rows - 1])
    check_rows(out[:rows - 1], want, "f16")
    assert not out[rows - 1].any() and not out[n - 1].any() and out[n - 2].any()
    width = call([0, 0], rows - 1, cu)[1]
    for c in (cu, None):
        out, _ = call([0, width - 1], rows, c)
        assert out[:rows].any(-1).all() and out[rows].any() and not out[rows + 1:].any()
        out, _ = call([width, 2**31 - 1], rows, c)
        assert not out.any()


def test_cache_attention_over_long_histories(db):
    """9000 keys of one head for one token: more parts than the join takes at a time; 3000 keys under a chunk of rows: more
    blocks than the many-row kernel keeps scales of."""
    gen, Hk, group = _gen(71), 1, 4
    for dtype in TYPES:
        for n, rows in ((9000, 1), (9001, 3), (3000, 40), (2990, 200)):
            k, v = (_randn(gen, n, Hk, 128, dtype=TYPES[dtype]) for _ in range(2))
            q = _randn(gen, rows, Hk * group, 128, dtype=TYPES[dtype])
            out, want = cached_rows(db, dtype, k, v, q, before=n - rows)
            check_rows(out, want, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_delta_thousands_of_tokens(db, dtype):
    """129 chunks under a slow decay.  To the 4e-6 of the state's RMS that one chunk may cost (see check_delta) come the
    roundings of 129 hand-overs, 2^-23 of the row's largest value (4 x RMS) each and at random: sqrt(129) 2^-21 / sqrt(12) =
    1.6e-6.  6e-6 and 6e-5 are allowed."""
    gen, Hk, Hv, T = _gen(81), 1, 2, 8229
    q, k, v, g, beta = delta_inputs(gen, T, Hk, Hv, TYPES[dtype], decay=0.001)
    s = _randn(gen, 1, Hv, 128, 128, scale=0.3)
    out, state = db.gated_delta(q, k, v, g, beta, state=s)
    want, want_state = delta_ref(q, k, v, g, beta, [T], s, 128 ** -0.5, 1e-6)
    err = (out.double().cpu() - want).abs()
    rms = want.square().mean().sqrt().item()
    assert torch.all(err <= 2 * EPS16[dtype] * (want.abs() + rms)), float((err / (want.abs() + rms)).max())
    d = state.double().cpu() - want_state
    srms = want_state.square().mean().sqrt().item()
    assert d.square().mean().sqrt().item() <= 6e-6 * srms and d.abs().max().item() <= 6e-5 * srms


CAPTURE = """
import sys
sys.path.insert(0, {root!r})
import torch, decisive_b200 as db
gen = torch.Generator("cuda").manual_seed(1)
B, Hk, Hq, V = 2, 2, 8, 5000
def randn(*shape): return torch.randn(shape, generator=gen, device="cuda").bfloat16()
def inputs(T):
    q, k, v = randn(B * T, Hq, 128), randn(B * T, Hk, 128), randn(B * T, Hk, 128)
    return [q, k, v, -torch.rand(B * T, Hq, generator=gen, device="cuda"), torch.rand(B * T, Hq, generator=gen, device="cuda"),
            randn(B, V)]
def state():
    c = db.KvCache8.allocate(B, 20, 10, Hk, torch.bfloat16)
    return [c, torch.zeros(B, Hq, 128, 128, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda"),
            torch.randint(V, (B, 7), generator=torch.Generator("cuda").manual_seed(2), device="cuda", dtype=torch.int32)]
def step(x, s, T):
    q, k, v, g, beta, logits = x
    db.kv8_append(s[0], k, v, s[2])
    a = db.kv8_attention(s[0], q, s[2])
    d, _ = db.gated_delta(k, k, q, g, beta, items=B, state=s[1], state_out=s[1])
    r = db.logit_rules(logits, s[3], repetition=torch.full((B,), 1.5, device="cuda"))
    s[2].add_(T)
    return [a, d, *r]
plan = [(40, [inputs(40) for _ in range(2)]), (1, [inputs(1) for _ in range(3)])]
eager, captured = state(), state()
torch.cuda.synchronize()
for T, steps in plan:
    hold = [x.clone() for x in steps[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # the first calls of this process
        got = step(hold, captured, T)
    for x in steps:
        for a, b in zip(hold, x):
            a.copy_(b)
        graph.replay()
        want = step(x, eager, T)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
assert torch.equal(eager[1], captured[1]) and torch.equal(eager[2], captured[2])
assert db.device_error_word() == 0
print("captured")
"""


def test_calls_can_be_captured(db):
    """A process whose first calls are captured in a CUDA graph; replays with other inputs, lengths and states are what
    calls outside a graph give."""
    r = subprocess.run([sys.executable, "-c", CAPTURE.format(root=ROOT)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("V,H,B", [(786432, 70000, 1), (786432, 100, 3), (600001, 65536, 2), (400000, 65535, 5)])
def test_rules_largest_vocabularies(db, V, H, B):
    """The largest vocabularies, with histories on both sides of what 16-bit counters hold, one id throughout a row."""
    gen = _gen(V + H)
    x = _randn(gen, B, V, scale=3.0)
    hist = torch.randint(0, V, (B, H), generator=gen, device="cuda", dtype=torch.int32)
    hist[0] = V - 1
    rho, pres, freq = (torch.rand(B, generator=gen, device="cuda") + o for o in (0.7, 0.1, 0.1))
    mask = torch.randint(-2**31, 2**31 - 1, (B, (V + 31) // 32), generator=gen, device="cuda").to(torch.int32)
    out, best, lse = db.logit_rules(x, hist, None, rho, pres, freq, mask=mask)
    want, wbest, wlse = rules_ref(x, hist, None, rho, pres, freq, None, None, mask)
    assert (out.cpu().numpy() == want).all() and best.tolist() == wbest
    assert np.allclose(lse.cpu().numpy(), np.array(wlse), rtol=2e-6, atol=1e-5)  # as in test_rules_match_the_definition
