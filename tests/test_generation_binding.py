"""CPU checks of what the generation entries and their Python wrappers do before any launch."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from decisive_b200 import build, _lib
    build.build()
    return _lib.load()


ONE = 4 * 128 * 128  # floats of a state of 4 heads


# Addresses in floats from a base that no device tensor has: every call is refused before it could launch anything.
@pytest.mark.parametrize("items,state,stride,state_out", [
    (3, 2 * ONE, 0, 0),         # a kept state that is a slot of the output
    (3, 0, 0, 0),               # ... the first one
    (2, ONE - 4, 0, 0),         # ... that ends inside
    (2, 0, 0, ONE - 4),         # ... that the output begins in
    (3, 0, ONE, ONE),           # states moved up by one item
    (3, ONE, ONE, 0),           # ... and down
    (2, 0, 2 * ONE, 0),         # every other state, packed
    (3, 0, 4 * ONE, 6 * ONE),   # the output lies over the third state of a wide stride
    (1, 0, ONE, 4), (1, 4, 0, 0),
])
def test_delta_refuses_states_that_meet(lib, items, state, stride, state_out):
    base = 1 << 20
    rc = lib.db_gated_delta(16, 16, 16, 1, 512, 512, 512, 16, 16, 4, 4, None, items, 4 * items, 4, 2, 4, 128, 1.0, -1.0,
                            base + 4 * state, stride, base + 4 * state_out, 16, 512, None, None)
    assert rc == -1 and lib.db_last_error_code() == b"INVALID_ARGUMENT"


class OnGpu1:
    """Stand-ins for tensors of device 1 while device 0 is current, and a library that notes what is current in each call."""

    def __init__(self, db, monkeypatch):
        torch = pytest.importorskip("torch")

        class Tensor(torch.Tensor):
            is_cuda = property(lambda self: True)

            def get_device(self):
                return 1

        class Device:
            def __init__(self, index):
                self.index = index

            def __enter__(self):
                outer.current.append(self.index)

            def __exit__(self, *_):
                outer.current.pop()

        class Library:
            def __getattr__(self, name):
                def entry(*args):
                    outer.calls.append((name, outer.current[-1], args[-1]))
                    return 64 if name.endswith("workspace_bytes") else 0
                return entry

        outer, self.current, self.calls = self, [0], []
        self.zeros = lambda dtype, *shape: torch.zeros(shape, dtype=dtype).as_subclass(Tensor)
        monkeypatch.setattr(db, "load", lambda: Library())
        monkeypatch.setattr(db, "_raw_stream", lambda device: 100 + device)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.current[-1], raising=False)
        monkeypatch.setattr(torch.cuda, "device", Device)


def test_calls_run_on_the_tensors_device(monkeypatch):
    import decisive_b200 as db
    torch = pytest.importorskip("torch")
    f16, f32, i32, i8 = torch.float16, torch.float32, torch.int32, torch.int8
    gpu = OnGpu1(db, monkeypatch)
    q = gpu.zeros(f16, 40, 2, 128)
    g = gpu.zeros(f32, 40, 2)
    db.gated_delta(q, q, q, g, g)
    cache = db.KvCache8(gpu.zeros(i8, 3, 2, 64, 128), gpu.zeros(f32, 3, 2), gpu.zeros(i8, 3, 2, 128, 64), gpu.zeros(f32, 3, 2),
                        gpu.zeros(f16, 1, 2, 64, 128), gpu.zeros(f16, 1, 2, 128, 64), gpu.zeros(i32, 1, 3))
    lengths = gpu.zeros(i32, 1)
    db.kv8_append(cache, q, q, lengths)
    db.kv8_attention(cache, q, lengths)
    db.kv8_read(cache, lengths, 10)
    db.logit_rules(gpu.zeros(f32, 2, 50))
    launches = [c for c in gpu.calls if not c[0].endswith("workspace_bytes")]
    assert [c[0] for c in launches] == ["db_gated_delta", "db_kv8_append", "db_kv8_attention", "db_kv8_read", "db_logit_rules"]
    assert len(gpu.calls) == 7 and all(c[1] == 1 for c in gpu.calls)  # workspaces are sized for the tensors' device too
    assert all(c[2] == 101 for c in launches) and gpu.current == [0]


def test_cache_follows_its_tensors(monkeypatch):
    """Calls read the addresses that the cache holds: a new page table is entered, nothing else can be swapped unseen."""
    import decisive_b200 as db
    torch = pytest.importorskip("torch")
    f16, f32, i32, i8 = torch.float16, torch.float32, torch.int32, torch.int8
    gpu = OnGpu1(db, monkeypatch)
    codes = lambda *s: gpu.zeros(i8, 3, 2, *s)  # noqa: E731
    scales, tail = gpu.zeros(f32, 3, 2), gpu.zeros(f16, 2, 2, 64, 128)
    cache = db.KvCache8(codes(64, 128), scales, codes(128, 64), scales, tail, tail.view(2, 2, 128, 64), gpu.zeros(i32, 2, 3))
    wider = gpu.zeros(i32, 2, 9)
    cache.page_table = wider
    assert cache.page_table is wider and cache.table_width == 9
    held = cache.ref._obj
    assert held.page_table == wider.data_ptr() and held.table_width == 9 and held.sequences == 2
    for bad in (gpu.zeros(i32, 3, 9), gpu.zeros(torch.int64, 2, 9), gpu.zeros(i32, 2, 18)[:, ::2], gpu.zeros(i32, 18)):
        with pytest.raises(ValueError):
            cache.page_table = bad
    assert cache.page_table is wider and held.page_table == wider.data_ptr()
    for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail", "table_width", "kv_heads", "dtype"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name))
