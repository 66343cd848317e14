"""GPU parity of the generation operators (gated delta rule, 8-bit paged cache and its attention, logit
rules) against plain float64 restatements of their definitions.

Tolerances, from the arithmetic: a 16-bit output carries one rounding of the result (2^-8 of a value for
bf16, 2^-11 for f16, both as bounds) and the kernels round nothing to fewer than 11 bits before it, so
outputs lie within 2 x the type's bound of the largest magnitude that a row's terms reach.  f32
states: sums of some 200 products in f32 (2^-24 each, growing with the root of their number) and, in
chunks, operands split into two f16 parts (2^-22): 4e-6 of the state's RMS, per element 4e-5."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS16 = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
FLT_MIN = float(np.finfo(np.float32).tiny)


@pytest.fixture(scope="module")
def db():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import decisive_b200 as d
    d.load()
    return d


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------------ gated delta rule
def delta_ref(q, k, v, g, beta, lens, state, scale, eps):
    """Token by token in float64 on the host."""
    q, k, v, g, beta = (x.double().cpu() for x in (q, k, v, g, beta))
    Hk, Hv = k.shape[1], v.shape[1]
    if eps is not None:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + eps)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + eps)
    q = (q * scale).repeat_interleave(Hv // Hk, 1)
    k = k.repeat_interleave(Hv // Hk, 1)
    out, states, r = torch.zeros_like(v), [], 0
    for b, n in enumerate(lens):
        S = torch.zeros(Hv, 128, 128, dtype=torch.float64)
        if state is not None:
            S = state[b if state.shape[0] > 1 else 0].double().cpu().clone()
        for t in range(r, r + n):
            S = S * torch.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - (S @ k[t][:, :, None])[..., 0])
            S = S + u[:, :, None] * k[t][:, None, :]
            out[t] = (S @ q[t][:, :, None])[..., 0]
        r += n
        states.append(S)
    return out, torch.stack(states)


def delta_inputs(gen, R, Hk, Hv, dt, strided=False, decay=0.3):
    if strided:
        w = _randn(gen, R, (2 * Hk + Hv + 1) * 128, dtype=dt)
        q, k, v = w[:, :Hk * 128], w[:, Hk * 128:2 * Hk * 128], w[:, 2 * Hk * 128:(2 * Hk + Hv) * 128]
        q, k, v = (x.unflatten(1, (-1, 128)) for x in (q, k, v))
    else:
        q, k, v = (_randn(gen, R, h, 128, dtype=dt) for h in (Hk, Hk, Hv))
    g = -decay * torch.nn.functional.softplus(_randn(gen, R, Hv))
    return q, k, v, g, torch.sigmoid(_randn(gen, R, Hv))


def check_delta(got, want, dtype):
    out, state = got
    ref_out, ref_state = want
    # a token's output is a sum over 128 keys of state times query: its scale is the rows' RMS
    err = (out.double().cpu() - ref_out).abs()
    rms = ref_out.square().mean().sqrt().item() if ref_out.numel() else 1.0
    assert torch.all(err <= 2 * EPS16[dtype] * (ref_out.abs() + rms)), float((err / (ref_out.abs() + rms)).max())
    d = state.double().cpu() - ref_state
    srms = ref_state.square().mean().sqrt().item()
    assert d.square().mean().sqrt().item() <= 4e-6 * srms + 1e-12
    assert d.abs().max().item() <= 4e-5 * srms + 1e-12


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,Hk,Hv,state", [(1, 1, 1, "none"), (1, 2, 6, "own"), (3, 2, 2, "shared"), (16, 1, 2, "own"),
                                           (17, 1, 3, "own"), (63, 2, 2, "none"), (64, 1, 2, "own"),
                                           (65, 2, 4, "shared"), (130, 1, 1, "own"), (385, 1, 2, "none")])
def test_delta_matches_the_recurrence(db, dtype, T, Hk, Hv, state):
    gen, B = _gen(T * 7 + Hv), 2
    q, k, v, g, beta = delta_inputs(gen, B * T, Hk, Hv, TYPES[dtype], strided=T % 2 == 1)
    s = None if state == "none" else _randn(gen, B if state == "own" else 1, Hv, 128, 128, scale=0.3)
    got = db.gated_delta(q, k, v, g, beta, items=B, state=s)
    check_delta(got, delta_ref(q, k, v, g, beta, [T] * B, s, 128 ** -0.5, 1e-6), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens", [[0, 5, 0, 1], [70, 1, 0, 129, 64], [200], [1, 2, 3, 4, 5, 6, 7]])
def test_delta_ragged(db, dtype, lens):
    gen, Hk, Hv = _gen(sum(lens)), 2, 4
    q, k, v, g, beta = delta_inputs(gen, sum(lens), Hk, Hv, TYPES[dtype])
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    s = _randn(gen, len(lens), Hv, 128, 128, scale=0.3)
    want = delta_ref(q, k, v, g, beta, lens, s, 128 ** -0.5, 1e-6)
    check_delta(db.gated_delta(q, k, v, g, beta, items=len(lens), cu_seqlens=cu, max_len=max(lens), state=s), want, dtype)
    check_delta(db.gated_delta(q, k, v, g, beta, items=len(lens), cu_seqlens=cu, state=s), want, dtype)  # no bound given
    # an item without rows passes its state on, bit for bit
    _, out_state = db.gated_delta(q, k, v, g, beta, items=len(lens), cu_seqlens=cu, state=s)
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.equal(out_state[b], s[b])


@pytest.mark.parametrize("T", [1, 70, 200])
def test_delta_in_place_and_split(db, T):
    """The state may be updated in place; a sequence cut in two gives what it gives whole."""
    gen, Hk, Hv = _gen(T), 1, 2
    q, k, v, g, beta = delta_inputs(gen, T, Hk, Hv, torch.bfloat16)
    s = _randn(gen, 1, Hv, 128, 128, scale=0.3)
    out, whole = db.gated_delta(q, k, v, g, beta, state=s)
    mine = s.clone()
    out2, same = db.gated_delta(q, k, v, g, beta, state=mine, state_out=mine)
    assert same is mine and torch.equal(mine, whole) and torch.equal(out, out2)
    c = T // 2
    if c:
        part = s.clone()
        db.gated_delta(q[:c], k[:c], v[:c], g[:c], beta[:c], state=part, state_out=part)
        db.gated_delta(q[c:], k[c:], v[c:], g[c:], beta[c:], state=part, state_out=part)
        rms = whole.double().square().mean().sqrt()
        assert (part - whole).double().square().mean().sqrt() <= 8e-6 * rms


@pytest.mark.parametrize("T", [2, 150])
def test_delta_resets_strong_decay_and_zeros(db, T):
    """g = -inf forgets all before the token; a decay far below f32's range; zero keys and values; beta 0 and 1."""
    gen, Hk, Hv = _gen(5), 1, 3
    q, k, v, g, beta = delta_inputs(gen, T, Hk, Hv, torch.float16)
    g[T // 2, 0] = -math.inf
    g[:, 1] = -200.0
    k[T // 3] = 0
    v[T // 2] = 0
    beta[:, 2] = 1.0
    beta[0] = 0.0
    s = _randn(gen, 1, Hv, 128, 128)
    got = db.gated_delta(q, k, v, g, beta, state=s)
    check_delta(got, delta_ref(q, k, v, g, beta, [T], s, 128 ** -0.5, 1e-6), "f16")


@pytest.mark.parametrize("T", [4, 100])
def test_delta_repeated_keys(db, T):
    """The same key at every token with beta near 1: the chunk's triangular system at its worst."""
    gen, Hk, Hv = _gen(6), 1, 2
    q, k, v, g, beta = delta_inputs(gen, T, Hk, Hv, torch.bfloat16, decay=0.001)
    k = k[:1].expand(T, -1, -1).contiguous()
    beta = torch.full_like(beta, 0.99)
    got = db.gated_delta(q, k, v, g, beta)
    check_delta(got, delta_ref(q, k, v, g, beta, [T], None, 128 ** -0.5, 1e-6), "bf16")


@pytest.mark.parametrize("T", [3, 90])
@pytest.mark.parametrize("size", [1e-3, 60.0])
def test_delta_without_norm(db, T, size):
    """Keys and queries as they come: small ones, and values in the thousands."""
    gen, Hk, Hv = _gen(7), 1, 2
    q, k, v, g, beta = delta_inputs(gen, T, Hk, Hv, torch.bfloat16)
    k = (k.float() / 128 ** 0.5).to(torch.bfloat16)  # near unit length, so that the recurrence is stable
    v = (v.float() * size * size).to(torch.bfloat16)
    q = (q.float() * 0.05 / size).to(torch.bfloat16)
    beta = beta * 0.5
    got = db.gated_delta(q, k, v, g, beta, norm_eps=None, scale=0.7)
    check_delta(got, delta_ref(q, k, v, g, beta, [T], None, 0.7, None), "bf16")


def test_delta_nan_stays_in_its_sequence(db):
    gen = _gen(8)
    q, k, v, g, beta = delta_inputs(gen, 180, 1, 2, torch.bfloat16)
    clean = db.gated_delta(q, k, v, g, beta, items=2)
    v2 = v.clone()
    v2[80, 0, 5] = math.nan  # item 0, head 0, value feature 5
    out, state = db.gated_delta(q, k, v2, g, beta, items=2)
    assert torch.equal(out[90:], clean[0][90:]) and torch.equal(state[1], clean[1][1])
    assert torch.equal(out[:90, 1], clean[0][:90, 1])
    assert torch.isnan(out[81:90, 0, 5]).all()


def test_delta_another_stream(db):
    gen = _gen(9)
    q, k, v, g, beta = delta_inputs(gen, 300, 2, 4, torch.bfloat16)
    want = db.gated_delta(q, k, v, g, beta)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [db.gated_delta(q, k, v, g, beta) for _ in range(3)]
    torch.cuda.synchronize()
    for o, s in got:
        assert torch.equal(o, want[0]) and torch.equal(s, want[1])


def test_delta_refusals(db):
    gen = _gen(1)
    q, k, v, g, beta = delta_inputs(gen, 6, 2, 4, torch.bfloat16)
    s = torch.zeros(2, 4, 128, 128, device="cuda")
    with pytest.raises(ValueError):
        db.gated_delta(q.half(), k, v, g, beta)
    with pytest.raises(ValueError):
        db.gated_delta(q, k, v, g.double(), beta)
    with pytest.raises(ValueError):
        db.gated_delta(q, k, v, g, beta, items=4)  # 6 rows do not divide
    with pytest.raises(ValueError):
        db.gated_delta(q[:, :, :64], k[:, :, :64], v[:, :, :64], g, beta)
    with pytest.raises(ValueError):
        db.gated_delta(q, k, v, g, beta, items=3, state=s)
    with pytest.raises(db.CudaError) as e:
        db.gated_delta(q, k, v[:, :3].contiguous(), g[:, :3].contiguous(), beta[:, :3].contiguous())
    assert e.value.code == "INVALID_ARGUMENT"
    one = torch.zeros(1, 4, 128, 128, device="cuda")
    lib = db.load()
    out = torch.empty_like(v)

    def raw(**kw):
        a = dict(ldq=256, items=2, rows=6, max_len=3, head_dim=128, state=one.data_ptr(), stride=0, state_out=s.data_ptr(),
                 dtype=2, q=q.data_ptr())
        a.update(kw)
        return lib.db_gated_delta(a["q"], k.data_ptr(), v.data_ptr(), a["dtype"], a["ldq"], 256, 512, g.data_ptr(),
                                  beta.data_ptr(), 4, 4, None, a["items"], a["rows"], a["max_len"], 2, 4, a["head_dim"],
                                  1.0, 1e-6, a["state"], a["stride"], a["state_out"], out.data_ptr(), 512, None, None)
    assert raw(head_dim=64) == -5 and raw(dtype=0) == -5
    assert raw(ldq=255) == -1 and raw(q=q.data_ptr() + 2) == -1 and raw(rows=7) == -1
    assert raw(state_out=one.data_ptr()) == -1  # one kept state for two items, updated in place
    assert raw(stride=4) == -1


# ------------------------------------------------------------------ 8-bit cache
class RefCache:
    """Every token in 16 bits, quantised block by block on demand."""

    def __init__(self, items, heads, dtype):
        self.k = [torch.zeros(0, heads, 128, dtype=dtype) for _ in range(items)]
        self.v = [torch.zeros(0, heads, 128, dtype=dtype) for _ in range(items)]

    def append(self, k, v, counts):
        r = 0
        for b, n in enumerate(counts):
            self.k[b] = torch.cat((self.k[b], k[r:r + n].cpu()))
            self.v[b] = torch.cat((self.v[b], v[r:r + n].cpu()))
            r += n

    @staticmethod
    def values(x):
        """f32 values as cached: full blocks through their codes (f32 arithmetic, as defined)."""
        n, parts = x.shape[0] // 64, []
        for i in range(n):
            blk = x[64 * i:64 * i + 64].float()
            s = (blk.abs().amax((0, 2), keepdim=True) * torch.tensor(1.0 / 127)).clamp(min=FLT_MIN)
            s[~torch.isfinite(s)] = math.nan
            code = torch.round(blk / s).clamp(-127, 127)
            parts.append(torch.where(torch.isnan(s), s, torch.nan_to_num(code) * s))
        parts.append(x[64 * n:].float())
        return torch.cat(parts)


def attention_ref(k, v, q, scale):
    """q [T, Hq, 128] at the end of k, v [n, Hk, 128], causal, float64."""
    T, Hq = q.shape[:2]
    n, Hk = k.shape[:2]
    r = Hq // Hk
    k, v, q = k.double(), v.double(), q.double()
    out = torch.zeros(T, Hq, 128, dtype=torch.float64)
    for i in range(T):
        seen = n - T + i + 1
        for h in range(Hq):
            s = (k[:seen, h // r] @ q[i, h]) * scale
            out[i, h] = torch.softmax(s, 0) @ v[:seen, h // r]
    return out


def new_cache(db, items, heads, dtype, tokens, gen, spare=3):
    """A cache with shuffled pages, uninitialised-looking contents and pages to spare."""
    width = tokens // 64 + 2
    pages = items * width + spare
    c = db.KvCache8.allocate(items, pages, width, heads, TYPES[dtype])
    c.page_table.copy_(torch.randperm(pages, generator=gen, device="cuda")[:items * width].view(items, width))
    c.k_codes.random_(-127, 127)
    c.v_codes.random_(-127, 127)
    c.k_scales.fill_(math.nan)
    c.v_scales.fill_(math.nan)
    c.k_tail.fill_(math.nan)
    c.v_tail.fill_(math.nan)
    return c


def check_attention(out, want, dtype):
    err = (out.double().cpu() - want).abs()
    # |softmax-weighted mean| terms: the values' magnitude near the row's, RMS as the floor
    rms = want.square().mean().sqrt().item()
    bound = 2 * EPS16[dtype] * (want.abs() + rms)
    assert torch.all(err <= bound), float((err / bound).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("Hq,Hk,steps", [
    (4, 1, [1, 1, 62, 1, 1, 1]), (8, 2, [130, 1, 1]), (2, 2, [64, 64, 1]), (10, 2, [700, 1, 3]), (8, 1, [65, 2, 61, 1]),
    (16, 1, [1, 127, 1]), (40, 1, [33, 1, 40]), (6, 2, [5, 200, 7])])
def test_cache_append_and_attention(db, dtype, Hq, Hk, steps):
    gen, B = _gen(Hq + sum(steps)), 2
    c = new_cache(db, B, Hk, dtype, sum(steps), gen)
    ref = RefCache(B, Hk, TYPES[dtype])
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    done = 0
    for T in steps:
        w = _randn(gen, B * T, (Hq + 2 * Hk) * 128, dtype=TYPES[dtype])
        q, k, v = (x.unflatten(1, (-1, 128)) for x in w.split((Hq * 128, Hk * 128, Hk * 128), 1))
        db.kv8_append(c, k, v, lengths)
        ref.append(k, v, [T] * B)
        out = db.kv8_attention(c, q, lengths, max_keys=done + T)
        wide = db.kv8_attention(c, q, lengths)
        lengths += T
        done += T
        got_k, got_v = db.kv8_read(c, lengths, done + 5)
        for b in range(B):
            k64, v64 = ref.values(ref.k[b]), ref.values(ref.v[b])
            assert torch.equal(got_k[b, :done].cpu(), k64) and torch.equal(got_v[b, :done].cpu(), v64)
            assert not got_k[b, done:].any() and not got_v[b, done:].any()
            rows = slice(b * T, (b + 1) * T)
            want = attention_ref(k64, v64, q[rows].cpu(), 128 ** -0.5)
            check_attention(out[rows], want, dtype)
            check_attention(wide[rows], want, dtype)
    assert db.device_error_word() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_cache_ragged_rows(db, dtype):
    gen, Hq, Hk = _gen(4), 8, 2
    counts = [[3, 0, 70, 1], [1, 64, 0, 130], [1, 1, 1, 1], [0, 63, 2, 5]]
    B = 4
    c = new_cache(db, B, Hk, dtype, 300, gen)
    ref = RefCache(B, Hk, TYPES[dtype])
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    for n in counts:
        at = np.concatenate([[0], np.cumsum(n)])
        cu = torch.tensor(at, dtype=torch.int32, device="cuda")
        R = int(at[-1])
        q, k, v = (_randn(gen, R, h, 128, dtype=TYPES[dtype]) for h in (Hq, Hk, Hk))
        db.kv8_append(c, k, v, lengths, cu_seqlens=cu, max_rows=max(n))
        ref.append(k, v, n)
        out = db.kv8_attention(c, q, lengths, cu_seqlens=cu, max_rows=max(n))
        lengths += torch.tensor(n, dtype=torch.int32, device="cuda")
        for b in range(B):
            if n[b]:
                rows = slice(at[b], at[b + 1])
                check_attention(out[rows], attention_ref(ref.values(ref.k[b]), ref.values(ref.v[b]), q[rows].cpu(), 128 ** -0.5), dtype)
    assert db.device_error_word() == 0


def test_cache_does_not_depend_on_the_split(db):
    """Token by token, in one piece, and in pieces: the same codes, scales and open block, bit for bit."""
    gen, Hk, n = _gen(11), 2, 200
    k, v = (_randn(gen, n, Hk, 128, dtype=torch.bfloat16) for _ in range(2))
    seen = []
    for pieces in ([n], [1] * n, [63, 1, 64, 72], [100, 100]):
        c = db.KvCache8.allocate(1, 4, 4, Hk, torch.bfloat16)
        lengths, at = torch.zeros(1, dtype=torch.int32, device="cuda"), 0
        for p in pieces:
            db.kv8_append(c, k[at:at + p], v[at:at + p], lengths)
            lengths += p
            at += p
        live = slice(0, n % 64)
        seen.append((c.k_codes, c.v_codes, c.k_scales, c.v_scales, c.k_tail[:, :, live], c.v_tail[:, :, :, live]))
    for other in seen[1:]:
        for x, y in zip(seen[0][:4], other[:4]):
            assert torch.equal(x[:3], y[:3])
        for x, y in zip(seen[0][4:], other[4:]):
            assert torch.equal(x, y)


def test_cache_extremes(db):
    """Zero blocks, one large value in a block, values near the type's limits, scores that overflow a
    plain exponential, a scale of zero."""
    gen, Hq, Hk, n = _gen(12), 4, 1, 150
    k, v = (_randn(gen, n, Hk, 128, dtype=torch.bfloat16) for _ in range(2))
    q = _randn(gen, 1, Hq, 128, dtype=torch.bfloat16)
    k[:64] = 0
    v[70, 0, 3] = 3e4
    v[64:66] = 1e-30
    v[130] = 1e20
    for qs, scale in ((1.0, 128 ** -0.5), (300.0, 1.0), (1e-20, 1e20), (1.0, 0.0)):
        c = new_cache(db, 1, Hk, "bf16", n, gen)
        lengths = torch.zeros(1, dtype=torch.int32, device="cuda")
        db.kv8_append(c, k, v, lengths)
        x = (q.float() * qs).to(torch.bfloat16)
        out = db.kv8_attention(c, x, lengths + n - 1, scale=scale)
        ref = RefCache(1, Hk, torch.bfloat16)
        ref.append(k, v, [n])
        check_attention(out, attention_ref(ref.values(ref.k[0]), ref.values(ref.v[0]), x.cpu(), scale), "bf16")


def test_cache_nonfinite_values(db):
    """A full block with a NaN or an infinity is NaN as a whole, for the rows that see it; in the open block
    the value reaches the rows that see its token; rows before are untouched."""
    gen, Hq, Hk = _gen(13), 4, 2
    n = 100
    q, k, v = (_randn(gen, n, h, 128, dtype=torch.float16) for h in (Hq, Hk, Hk))
    v[90, 0, 7] = math.inf  # open block, head 0
    k[95, 1, 0] = math.nan  # open block, head 1
    c = new_cache(db, 1, Hk, "f16", n, gen)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    db.kv8_append(c, k, v, zero)
    out = db.kv8_attention(c, q, zero)
    assert torch.isfinite(out[:90]).all() and torch.isfinite(out[:95, 2:]).all()
    assert (out[90:, :2, 7] == math.inf).all() and torch.isfinite(out[90:, :2, 8:]).all()
    assert torch.isnan(out[95:, 2:]).all()
    k[20, 0, 0] = -math.inf  # a full block now
    c = new_cache(db, 1, Hk, "f16", n, gen)
    db.kv8_append(c, k, v, zero)
    got_k, _ = db.kv8_read(c, zero + n, n)
    assert torch.isnan(got_k[0, :64, 0]).all() and torch.isfinite(got_k[0, :64, 1]).all()
    # the next block's rows of a later call do see it; a sequence beside it does not
    assert torch.isnan(db.kv8_attention(c, q, zero)[64:, :2]).all()


def test_cache_missing_pages_and_bad_lengths(db):
    """Tables and lengths that name nothing are skipped and noted, not followed."""
    gen, Hk = _gen(14), 1
    c = new_cache(db, 1, Hk, "f16", 200, gen)
    q, k, v = (_randn(gen, 128, 1, 128, dtype=torch.float16) for _ in range(3))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert db.device_error_word() == 0
    c.page_table[0, 0] = -1
    c.page_table[0, 1] = 1 << 30
    db.kv8_append(c, k, v, zero)
    out = db.kv8_attention(c, q, zero)
    assert not out.any()  # no key could be read
    assert db.device_error_word() == 0x10 and db.device_error_word() == 0
    c = new_cache(db, 1, Hk, "f16", 200, gen)
    before = [x.clone() for x in (c.k_codes, c.k_tail)]
    for bad in (-5, 2**31 - 1, c.page_table.shape[1] * 64):
        db.kv8_append(c, k[:1], v[:1], torch.full_like(zero, bad))
        db.kv8_attention(c, q[:1], torch.full_like(zero, bad))
        assert db.device_error_word() == 0x10
    assert torch.equal(before[0], c.k_codes)


def test_cache_refusals(db):
    gen = _gen(15)
    c = new_cache(db, 2, 2, "f16", 64, gen)
    k = _randn(gen, 2, 2, 128, dtype=torch.float16)
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        db.kv8_append(c, k.bfloat16(), k.bfloat16(), lengths)
    with pytest.raises(ValueError):
        db.kv8_append(c, k[:, :1], k[:, :1], lengths)
    with pytest.raises(ValueError):
        db.kv8_append(c, k, k, lengths.long())
    with pytest.raises(ValueError):
        db.KvCache8(c.k_codes, c.k_scales, c.v_codes.transpose(2, 3), c.v_scales, c.k_tail, c.v_tail, c.page_table)
    with pytest.raises(db.CudaError):
        db.kv8_attention(c, _randn(gen, 2, 3, 128, dtype=torch.float16), lengths)  # 3 heads over 2
    with pytest.raises(db.CudaError):
        db.kv8_append(c, k.repeat(2, 1, 1), k.repeat(2, 1, 1), lengths.repeat(2))  # more items than sequences
    with pytest.raises(ValueError):
        db.kv8_append(c, k[:, :, 1:], k[:, :, 1:], lengths)
    wide = _randn(gen, 2 * 260).half().view(2, 260)[:, :256].unflatten(1, (2, 128))
    with pytest.raises(db.CudaError):
        db.kv8_append(c, wide, wide, lengths)  # rows 260 apart do not start on 16 bytes
    db.kv8_append(c, k[:0], k[:0], lengths[:0])  # nothing to do


# ------------------------------------------------------------------ logit rules
def rules_ref(x, history, lens, rho, pres, freq, ids, vals, mask):
    """Row by row in f32, operation by operation as defined; the statistics in float64."""
    x = x.float().cpu().numpy().copy()
    B, V = x.shape
    best, lse = [], []
    for b in range(B):
        if history is not None:
            h = history[b].cpu().numpy()
            h = h[:len(h) if lens is None else max(0, min(int(lens[b]), len(h)))]
            h = h[(h >= 0) & (h < V)]
            c = np.bincount(h, minlength=V).astype(np.float32)
            one = np.float32
            r = one(rho[b].item()) if rho is not None else one(1)
            p = one(pres[b].item()) if pres is not None else one(0)
            f = one(freq[b].item()) if freq is not None else one(0)
            y = np.where(x[b] > 0, x[b] / r, x[b] * r) - (p + f * c)
            x[b] = np.where(c > 0, y, x[b])
        if ids is not None:
            for i, w in zip(ids[b].tolist(), vals[b].cpu().numpy()):
                if 0 <= i < V:
                    x[b, i] = np.float32(x[b, i] + w)
        if mask is not None:
            w = mask[b].cpu().numpy().view(np.uint32)
            v = np.arange(V)
            x[b][(w[v // 32] >> (v % 32)) & 1 == 0] = -np.inf
        z = x[b].astype(np.float64)
        top = np.nanmax(np.where(np.isnan(z), -np.inf, z))
        best.append(-1 if top == -np.inf else int(np.flatnonzero(z == top)[0]))
        if np.isnan(z).any():
            lse.append(math.nan)
        elif not np.isfinite(top):
            lse.append(top)
        else:
            lse.append(top + math.log(np.exp(z - top).sum()))
    return x, best, lse


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,V,H,K", [(1, 1, 1, 1), (2, 33, 40, 3), (3, 1000, 0, 0), (2, 4099, 500, 64), (4, 32000, 2048, 300),
                                     (2, 151936, 576, 8), (1, 128100, 5000, 1024), (300, 97, 5, 2)])
def test_rules_match_the_definition(db, dtype, B, V, H, K):
    gen = _gen(V + H)
    x = _randn(gen, B, V, scale=3.0, dtype=dtype)
    hist = torch.randint(-2, V + 2, (B, H), generator=gen, device="cuda", dtype=torch.int32) if H else None
    lens = torch.randint(0, H + 2, (B,), generator=gen, device="cuda", dtype=torch.int32) if H else None
    rho, pres, freq = (torch.rand(B, generator=gen, device="cuda") + o for o in (0.7, -0.2, -0.1))
    ids = torch.randint(-1, V + 1, (B, K), generator=gen, device="cuda", dtype=torch.int32) if K else None  # repeats
    vals = _randn(gen, B, K) if K else None
    mask = torch.randint(-2**31, 2**31 - 1, (B, (V + 31) // 32), generator=gen, device="cuda").to(torch.int32)
    if B > 1:
        mask[1] = 0  # nothing allowed
    out, best, lse = db.logit_rules(x, hist, lens, rho, pres, freq, ids, vals, mask)
    want, wbest, wlse = rules_ref(x, hist, lens, rho, pres, freq, ids, vals, mask)
    assert np.array_equal(out.cpu().numpy(), want)
    assert best.tolist() == wbest
    # sums of positive terms in f32 and a logarithm: 1e-5 absolute covers 2^-24 x the terms' depth
    assert np.allclose(lse.cpu().numpy(), np.array(wlse, np.float64), rtol=2e-6, atol=1e-5, equal_nan=True)


def test_rules_ties_infinities_and_nan(db):
    V = 5000
    x = torch.zeros(6, V, device="cuda")
    x[0, [77, 4000, 3]] = 2.5           # ties: the lowest id
    x[1] = -math.inf                    # nothing left
    x[2, 4321] = math.inf               # one certain token
    x[3, 10] = math.nan                 # a NaN is never the best
    x[3, 20] = 1.0
    x[4] = torch.finfo(torch.float32).min  # the type's lowest value is a value
    x[5, 9] = math.nan
    mask = torch.full((6, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    mask[5, 0] &= ~(1 << 9)             # a NaN that is masked does not count
    out, best, lse = db.logit_rules(x, mask=mask)
    assert best.tolist() == [3, -1, 4321, 20, 0, 0]
    got = lse.tolist()
    assert got[1] == -math.inf and got[2] == math.inf and math.isnan(got[3])
    assert got[4] == pytest.approx(torch.finfo(torch.float32).min) and got[5] == pytest.approx(math.log(V - 1), rel=1e-6)
    assert out[5, 9].item() == -math.inf and math.isnan(out[3, 10].item())


def test_rules_strides_and_in_place(db):
    gen = _gen(3)
    for V, ld in ((1000, 1003), (1000, 1008), (77, 80)):
        base = _randn(gen, 4, ld)
        x = base[:, :V]
        hist = torch.randint(0, V, (4, 30), generator=gen, device="cuda", dtype=torch.int32)
        rho = torch.full((4,), 1.5, device="cuda")
        want, best, lse = db.logit_rules(x.contiguous(), hist, repetition=rho)
        got, best2, lse2 = db.logit_rules(x, hist, repetition=rho)
        assert torch.equal(got, want) and torch.equal(best, best2) and torch.allclose(lse, lse2, atol=1e-5)
        keep = base[:, V:].clone()
        same, _, _ = db.logit_rules(x, hist, repetition=rho, out=x)
        assert same is x and torch.equal(x, want) and torch.equal(base[:, V:], keep)


def test_rules_refusals(db):
    x = torch.zeros(2, 100, device="cuda")
    ids = torch.zeros(2, 1025, dtype=torch.int32, device="cuda")
    with pytest.raises(db.CudaError) as e:
        db.logit_rules(x, bias_ids=ids, bias_values=torch.zeros(2, 1025, device="cuda"))
    assert e.value.code == "UNSUPPORTED"
    with pytest.raises(db.CudaError):
        db.logit_rules(x, bias_ids=ids[:, :4].contiguous())  # ids without values
    with pytest.raises(ValueError):
        db.logit_rules(x.double())
    with pytest.raises(ValueError):
        db.logit_rules(x, mask=torch.zeros(2, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        db.logit_rules(x, history=torch.zeros(2, 5, dtype=torch.int64, device="cuda"))
    with pytest.raises(db.CudaError):
        db.logit_rules(torch.zeros(1, 800000, device="cuda"))
