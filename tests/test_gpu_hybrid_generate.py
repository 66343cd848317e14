"""The generation operators together, as examples/hybrid_generate.py runs them, and the cache where its pages lie far
out."""
import importlib.util
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def hybrid():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    spec = importlib.util.spec_from_file_location("hybrid_generate", os.path.join(ROOT, "examples", "hybrid_generate.py"))
    m = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = m  # (dataclasses look their module up)
    spec.loader.exec_module(m)
    return m


def _prompts(vocab, lengths):
    rng = torch.Generator().manual_seed(5)
    return [torch.randint(vocab, (n,), generator=rng).tolist() for n in lengths]


def test_generates_under_the_rules(hybrid):
    s = hybrid.Sizes(layers=4, hidden=256, vocab=1000)
    prompts = _prompts(s.vocab, (130, 17, 1))
    mask = torch.full((3, 32), 0x11111111, dtype=torch.int32, device="cuda")  # every fourth id
    runs = [hybrid.generate(hybrid.Hybrid(s, 3, 140), prompts, 10, mask, repetition=1.0, presence=1e4, frequency=0.0)
            for _ in range(2)]
    ids, logs = runs[0]
    assert torch.equal(ids, runs[1][0]) and torch.equal(logs, runs[1][1])  # nothing depends on the order of atomics
    assert ids.shape == (3, 10) and bool((ids % 4 == 0).all()) and bool((logs <= 0).all())
    for row, prompt in zip(ids.tolist(), prompts):  # a penalty above all logits: no id twice, none of the prompt's
        assert len(set(row)) == len(row) and not set(row) & set(prompt)


def test_a_prompt_at_once_is_its_tokens_one_by_one(hybrid):
    """40 tokens (no block fills up, so neither way reads codes).  The ways differ by roundings to bf16: 8 layers of some four
    of 2^-9 each, as good as random: 2^-9 sqrt(32) = 0.011 of the logits' RMS; 0.05 is allowed."""
    s = hybrid.Sizes(vocab=1000)
    tokens = torch.tensor(_prompts(s.vocab, (40,))[0], device="cuda")
    at_once, steps = hybrid.Hybrid(s, 1, 64), hybrid.Hybrid(s, 1, 64)
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    a = at_once.forward(tokens, 40, cu, 40)
    for i in range(40):
        b = steps.forward(tokens[i:i + 1], i + 1)
    assert bool(torch.isfinite(a).all())
    assert ((a - b).square().mean().sqrt() / b.square().mean().sqrt()).item() < 0.05
    for x, y in zip(at_once.states, steps.states):
        if torch.is_tensor(x):
            assert ((x - y).square().mean().sqrt() / y.square().mean().sqrt()).item() < 0.05


@pytest.mark.parametrize("v_heads", [1, 5, 9])
def test_heads_that_share_a_key_head(v_heads):
    """Many chunks, so that one CTA prepares all value heads of a key head, in batches: the same products in the same order as
    with a key head for each, so the same bits."""
    import decisive_b200 as db
    rng, rows = torch.Generator("cuda").manual_seed(v_heads), 64 * 600 + 7
    q, k = (torch.randn(rows, 1, 128, generator=rng, device="cuda").bfloat16() for _ in range(2))
    v = torch.randn(rows, v_heads, 128, generator=rng, device="cuda").bfloat16()
    g = -torch.rand(rows, v_heads, generator=rng, device="cuda")
    beta = torch.rand(rows, v_heads, generator=rng, device="cuda")
    cu = torch.tensor([0, 64 * 300 + 5, rows], dtype=torch.int32, device="cuda")
    shared = db.gated_delta(q, k, v, g, beta, items=2, cu_seqlens=cu)
    own = db.gated_delta(q.expand(-1, v_heads, -1).contiguous(), k.expand(-1, v_heads, -1).contiguous(), v, g, beta, items=2,
                         cu_seqlens=cu)
    for x, y in zip(shared, own):
        assert bool(torch.isfinite(x).all()) and torch.equal(x, y)


@pytest.mark.parametrize("rows", [1, 40])  # per kv head: the two forms of the attention
def test_pages_past_32_bits(rows):
    """A page whose first code lies 2.4 billion bytes into the pool reads as page 0 does."""
    import decisive_b200 as db
    pages = 300000
    rng = torch.Generator("cuda").manual_seed(9)
    k, v = (torch.randn(64 + rows, 1, 128, generator=rng, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(rows, 1, 128, generator=rng, device="cuda").bfloat16()
    outs = []
    for page, pool in ((0, 1), (pages - 1, pages)):
        c = db.KvCache8.allocate(1, pool, 2, 1, torch.bfloat16)
        c.page_table[:] = torch.tensor([[page, -1]], dtype=torch.int32)
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        db.kv8_append(c, k[:64], v[:64], zero)
        db.kv8_append(c, k[64:], v[64:], zero + 64)
        outs.append((db.kv8_attention(c, q, zero + 64), *db.kv8_read(c, zero + 64 + rows, 64 + rows)))
        assert bool(c.k_codes[page].any()) and bool(c.v_codes[page].any())
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_cache_and_rules_on_their_stream():
    """Calls go to the current stream: inputs that another stream still writes are waited for."""
    import decisive_b200 as db
    side = torch.cuda.Stream()
    rng = torch.Generator("cuda").manual_seed(3)
    k, v, q = (torch.randn(70, 2, 128, generator=rng, device="cuda").half() for _ in range(3))
    logits = torch.randn(3, 5000, generator=rng, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    c = db.KvCache8.allocate(1, 2, 2, 2, torch.float16)
    db.kv8_append(c, k, v, zero)
    want = (db.kv8_attention(c, q, zero), *db.logit_rules(logits))
    torch.cuda.synchronize()
    c = db.KvCache8.allocate(1, 2, 2, 2, torch.float16)
    late = torch.zeros_like(logits)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            x = x @ x * 1e-4  # a while
        late.copy_(logits)
        db.kv8_append(c, k, v, zero)
        got = (db.kv8_attention(c, q, zero), *db.logit_rules(late))
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
