"""CPU checks of the generation entries (gated delta rule, 8-bit cache, logit rules): constants of header and binding
agree, sizes of workspaces, and what is refused before any device work."""
import ctypes as C
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from decisive_b200 import build, _lib
    build.build()
    return _lib.load()


def _code(lib):
    return lib.db_last_error_code().decode()


def test_constants_match_the_header():
    import decisive_b200 as db
    text = open(os.path.join(ROOT, "include", "decisive_b200.h")).read()
    defined = {k: int(v) for k, v in re.findall(r"#define (DB_KV8_BLOCK|DB_DELTA_STEP_TOKENS) (\d+)", text)}
    assert defined == {"DB_KV8_BLOCK": db.KvCache8.BLOCK, "DB_DELTA_STEP_TOKENS": db.DELTA_STEP_TOKENS}


def test_cache_struct_matches_the_header():
    from decisive_b200 import _lib
    text = open(os.path.join(ROOT, "include", "decisive_b200.h")).read()
    body = re.search(r"typedef struct db_kv8_cache \{(.*?)\} db_kv8_cache;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [re.sub(r"[*\s]", "", n) for line in body.split(";") if line.strip()
             for n in re.sub(r"^\s*(const\s+)?\w+\s", "", line.strip()).split(",")]
    assert names == [f[0] for f in _lib.KvCache8._fields_]
    assert C.sizeof(_lib.KvCache8) == 7 * C.sizeof(C.c_void_p) + 6 * 4


def test_delta_workspace(lib):
    size = lib.db_gated_delta_workspace_bytes
    assert size(4, 64, 16, 2, 4, 1) == 0  # single tokens and short items need none
    f16, bf16 = size(4, 4096, 1024, 2, 4, 1), size(4, 4096, 1024, 2, 4, 2)
    assert 0 < f16 < bf16                 # bf16 rows are kept as f16 beside the triangles
    assert size(4, 8192, 2048, 2, 4, 1) > f16
    assert size(0, 0, 0, 2, 4, 1) == size(-1, 5, 5, 1, 1, 1) == 0


def _delta(lib, dtype=1, items=1, rows=4, max_len=4, hk=2, hv=4, head_dim=128, ptr=16, ld=512, ldg=4, state=None,
           stride=0, state_out=None, cu=None, workspace=None):
    return lib.db_gated_delta(ptr, ptr, ptr, dtype, ld, ld, ld, ptr, ptr, ldg, ldg, cu, items, rows, max_len, hk, hv,
                              head_dim, 1.0, -1.0, state, stride, state_out, ptr, ld, workspace, None)


@pytest.mark.parametrize("change", [
    dict(items=-1), dict(items=65536), dict(rows=5), dict(max_len=5, cu=16), dict(hk=3), dict(hk=0), dict(ptr=None),
    dict(ptr=24), dict(ld=256), dict(ld=516), dict(ldg=3), dict(state=16, stride=4), dict(state=16, stride=65538),
    dict(items=2, rows=8, state=16, state_out=16), dict(rows=64, max_len=64)])
def test_delta_refuses(lib, change):
    assert _delta(lib, **change) == -1 and _code(lib) == "INVALID_ARGUMENT"


@pytest.mark.parametrize("change", [dict(head_dim=64), dict(dtype=0), dict(dtype=3)])
def test_delta_does_not_support(lib, change):
    assert _delta(lib, **change) == -5 and _code(lib) == "UNSUPPORTED"


def test_delta_without_items_is_nothing(lib):
    assert _delta(lib, items=0, rows=0, max_len=0) == 0


def _cache(**change):
    from decisive_b200 import _lib
    fields = dict(k_codes=16, k_scales=16, v_codes=16, v_scales=16, k_tail=16, v_tail=16, page_table=16, pages=8, table_width=4,
                  sequences=2, kv_heads=2, head_dim=128, dtype=2)
    fields.update(change)
    return _lib.KvCache8(**fields)


BAD_CACHES = [dict(kv_heads=0), dict(pages=-1), dict(table_width=-1), dict(table_width=1 << 26), dict(sequences=1),
              dict(k_codes=24), dict(v_tail=None), dict(page_table=None), dict(k_scales=None)]


@pytest.mark.parametrize("change", BAD_CACHES)
def test_cache_calls_refuse_a_bad_cache(lib, change):
    c = C.byref(_cache(**change))
    for rc in (lib.db_kv8_append(c, 16, 256, 16, 256, 16, None, 2, 2, 1, None),
               lib.db_kv8_attention(c, 16, 512, 16, None, 2, 2, 1, 64, 4, 1.0, 16, 512, 16, None),
               lib.db_kv8_read(c, 16, 2, 64, 16, 16, None)):
        assert rc == -1 and _code(lib) == "INVALID_ARGUMENT"


@pytest.mark.parametrize("change", [dict(head_dim=64), dict(dtype=0)])
def test_cache_calls_do_not_support(lib, change):
    c = C.byref(_cache(**change))
    assert lib.db_kv8_append(c, 16, 256, 16, 256, 16, None, 2, 2, 1, None) == -5 and _code(lib) == "UNSUPPORTED"


def test_cache_calls_refuse_bad_rows(lib):
    c = C.byref(_cache())
    for rc in (lib.db_kv8_append(None, 16, 256, 16, 256, 16, None, 2, 2, 1, None) + 4,  # no cache: UNSUPPORTED, -5
               lib.db_kv8_append(c, 16, 256, 16, 256, 16, None, 2, 3, 1, None),      # rows are not items x max_rows
               lib.db_kv8_append(c, 16, 128, 16, 256, 16, None, 2, 2, 1, None),      # short rows
               lib.db_kv8_append(c, 24, 256, 16, 256, 16, None, 2, 2, 1, None),      # unaligned
               lib.db_kv8_attention(c, 16, 512, 16, None, 2, 2, 1, 64, 3, 1.0, 16, 512, 16, None),
               lib.db_kv8_attention(c, 16, 512, 16, None, 2, 2, 1, 0, 4, 1.0, 16, 512, 16, None),
               lib.db_kv8_attention(c, 16, 512, 16, None, 2, 2, 1, 64, 4, 1.0, 16, 516, 16, None),
               lib.db_kv8_read(c, 16, 2, -1, 16, 16, None), lib.db_kv8_read(c, 16, 2, 64, None, 16, None)):
        assert rc == -1


def _rules(lib, dtype=0, ld=64, rows=2, vocab=64, history=None, ldh=0, lens=None, cols=0, ids=None, values=None, biases=0,
           mask=None, ldm=0, logits=16, out=32, ldo=64):
    return lib.db_logit_rules(logits, dtype, ld, rows, vocab, history, ldh, lens, cols, None, None, None, ids, values,
                              biases, mask, ldm, out, ldo, None, None, None)


@pytest.mark.parametrize("change", [
    dict(rows=-1), dict(rows=65536), dict(vocab=0), dict(ld=63), dict(ldo=63), dict(logits=None), dict(out=None),
    dict(mask=16, ldm=1), dict(history=16, ldh=3, cols=4), dict(lens=16), dict(ids=16, biases=1), dict(biases=-1),
    dict(dtype=2, out=16)])
def test_rules_refuse(lib, change):
    assert _rules(lib, **change) == -1 and _code(lib) == "INVALID_ARGUMENT"


@pytest.mark.parametrize("change", [dict(dtype=3), dict(vocab=786433, ld=786433, ldo=786433),
                                    dict(ids=16, values=16, biases=1025)])
def test_rules_do_not_support(lib, change):
    assert _rules(lib, **change) == -5 and _code(lib) == "UNSUPPORTED"


def test_empty_calls_are_nothing(lib):
    assert _rules(lib, rows=0) == 0
    c = C.byref(_cache())
    assert lib.db_kv8_append(c, None, 0, None, 0, None, None, 0, 0, 0, None) == 0
    assert lib.db_kv8_read(c, 16, 2, 0, None, None, None) == 0
