"""decisive_b200: B200 (sm_100a) backend for decisive's quantised projection path.

Two layers, both thin over the C ABI of libdecisive_b200.so (include/decisive_b200.h):

* kernel level -- torch-tensor wrappers of the group-64 quantiser, weight packer, grouped GEMM
  (tensor-core and GEMV paths), fused MLP, attention and dequantisation.  torch supplies device
  memory and streams only; every computation runs in this library's CUDA kernels.
* model level -- ``Model`` / ``Cache`` / ``Cancellation`` / ``Error`` mirroring the reference's
  ``inference`` module (src/inference/mod.rs:17-273): ``predict`` and ``predict_batch`` with the
  same error codes, cache ownership and cancellation rules.
"""
from __future__ import annotations

import ctypes as C
import json
from dataclasses import dataclass, field
from operator import attrgetter

from . import _lib
from ._lib import CudaError, check, load

GROUP = 64
CODES_NATURAL, CODES_GEMV, CODES_TC, CODES_DQ = 0, 1, 2, 3
DTYPES = {"float32": 0, "float16": 1, "bfloat16": 2}


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _stream(stream=None):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def padded(k: int) -> int:
    return (k + GROUP - 1) // GROUP * GROUP


def scale_stride(n: int) -> int:
    """Row stride of scale arrays: roundup(n, 128) (db_scale_row_stride)."""
    return (n + 127) // 128 * 128


# ------------------------------------------------------------------ kernel level
def quantize_activations(x, bits: int = 8, layout: int = CODES_TC, sums: bool = False, nonfinite=None):
    """int8::Matrix::prepare (int8.rs:178-202) on the GPU -> (codes, scales [G, M], sums [G, M] | None)."""
    import torch
    assert x.is_cuda and x.dim() == 2
    M, K = x.shape
    Kp = padded(K)
    G = Kp // GROUP
    dt = torch.float16 if layout in (CODES_TC, CODES_DQ) else torch.int8
    codes = torch.zeros((M, Kp), dtype=dt, device=x.device)
    lds = scale_stride(max(M, 1))
    scales = torch.zeros((G, lds), dtype=torch.float32, device=x.device)
    s = torch.zeros((G, lds), dtype=torch.int32, device=x.device) if sums else None
    check(load().db_quantize_activations_g64(_ptr(x), DTYPES[str(x.dtype).split(".")[1]], x.stride(0), M, K, bits,
                                             _ptr(codes), layout, Kp, _ptr(scales), _ptr(s), lds,
                                             _ptr(nonfinite), _stream()))
    return codes, scales, s


def pack_weights(bf16, bits: int = 4):
    """Absmax group-64 weight quantiser (int8.rs:51-152, packed.rs:31-56): bf16 [N, K] (as int16/uint16
    bits or torch.bfloat16) -> (codes, scales [G, N])."""
    import torch
    N, K = bf16.shape
    Kp = padded(K)
    codes = torch.empty((N, Kp * bits // 8), dtype=torch.uint8, device=bf16.device)
    scales = torch.empty((Kp // GROUP, scale_stride(N)), dtype=torch.float32, device=bf16.device)
    check(load().db_pack_weights_g64(_ptr(bf16), N, K, bits, _ptr(codes), _ptr(scales), _stream()))
    return codes, scales


def import_packed(packed, N: int, K: int, bits: int):
    import torch
    codes = torch.empty((N, K * bits // 8), dtype=torch.uint8, device=packed.device)
    scales = torch.empty((K // GROUP, scale_stride(N)), dtype=torch.float32, device=packed.device)
    check(load().db_import_packed(_ptr(packed), N, K, bits, _ptr(codes), _ptr(scales), _stream()))
    return codes, scales


def export_packed(codes, scales, N: int, K: int, bits: int):
    import torch
    out = torch.empty(N * (K // GROUP) * (GROUP * bits // 8 + 4), dtype=torch.uint8, device=codes.device)
    check(load().db_export_packed(_ptr(codes), _ptr(scales), N, K, bits, _ptr(out), _stream()))
    return out


def dequant_rows(codes, scales, N: int, K: int, bits: int, ids=None):
    import torch
    T = N if ids is None else ids.numel()
    out = torch.empty((T, K), dtype=torch.float32, device=codes.device)
    check(load().db_dequant_rows_g64(_ptr(codes), _ptr(scales), N, K, bits, _ptr(ids), T, _ptr(out), K, _stream()))
    return out


class GemmConfig(C.Structure):
    """db_gemm_config: tile width (0 = default, 64, 128, 256), persistent grid cap (0 = all SMs) and
    CTA pairing (1 = clusters of two CTAs with M = 256 MMAs).  The tuner's candidate space."""
    _fields_ = [("block_n", C.c_int), ("max_ctas", C.c_int), ("pair_ctas", C.c_int)]


def gemm(a_codes, layout, sa, w_codes, sw, M, N, K, bits, fused=True, a_sums=None, residual=None, nonfinite=None,
         config=None):
    """Matrix::apply_prepared (int8.rs:229-288) on prepared activations -> y f32 [M, N].
    config: optional GemmConfig (tile configuration of the tensor-core path).  CODES_DQ: a_codes are
    the dequantised f16 activations (sa may be None); the kind::f16 full-K GEMM (tolerance numerics)."""
    import torch
    y = residual if residual is not None else torch.empty((M, N), dtype=torch.float32, device=w_codes.device)
    cfg = C.byref(config) if config is not None else None
    check(load().db_gemm_g64_config(_ptr(a_codes), layout, a_codes.stride(0), _ptr(sa), _ptr(a_sums),
                                    sa.stride(0) if sa is not None else 0,
                                    _ptr(w_codes), _ptr(sw), M, N, K, bits, int(fused), int(residual is not None),
                                    _ptr(y), N, _ptr(nonfinite), cfg, _stream()))
    return y


def decima_quantize_weights(w, block: int = 32):
    """decima::int8::Matrix::new (W8, decima/int8.rs:106-151): f32 [N, K] device tensor ->
    (codes uint8 [N, Kp], scales f32 [ceil(K/block), scale_stride(N)])."""
    import torch
    N, K = w.shape
    Kp = -(-K // GROUP) * GROUP
    codes = torch.zeros((N, Kp), dtype=torch.uint8, device=w.device)
    scales = torch.empty((-(-K // block), scale_stride(N)), dtype=torch.float32, device=w.device)
    check(load().db_decima_quantize_weights(_ptr(w), N, K, block, _ptr(codes), _ptr(scales), _stream()))
    return codes, scales


def decima_quantize_activations(x, block: int = 32, layout: int = CODES_TC):
    """The activation fill of decima Matrix::apply_with_rows: f32 [M, K] -> (codes, scales, nonfinite flag)."""
    import torch
    M, K = x.shape
    Kp = -(-K // GROUP) * GROUP
    dt = torch.float16 if layout == CODES_TC else torch.int8
    codes = torch.zeros((M, Kp), dtype=dt, device=x.device)
    scales = torch.empty((-(-K // block), scale_stride(M)), dtype=torch.float32, device=x.device)
    flag = torch.zeros(1, dtype=torch.int32, device=x.device)
    check(load().db_decima_quantize_activations(_ptr(x), M, K, block, _ptr(codes), layout, Kp, _ptr(scales),
                                                scales.stride(0), _ptr(flag), _stream()))
    return codes, scales, flag


def decima_linear(x, w_codes, w_scales, N: int, block: int = 32, fused: bool = True, bias=None):
    """decima Matrix::apply_with_rows, WeightsActivations mode: y [M, N] = W8A8 grouped GEMM + bias."""
    import torch
    M, K = x.shape
    ws = torch.empty(load().db_decima_workspace_bytes(M, K, block), dtype=torch.uint8, device=x.device)
    y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    check(load().db_decima_linear(_ptr(x), M, K, _ptr(w_codes), _ptr(w_scales), N, block, int(fused), _ptr(bias),
                                  _ptr(y), _ptr(ws), _stream()))
    return y


def decima_linear_w8a32(x, w_codes, w_scales, N: int, block: int = 32, fused: bool = True, bias=None):
    """decima Matrix::apply_with_rows, Weights mode: y [M, N] = f32 x times the int8 weight codes
    (decoded with their block scales) + bias."""
    import torch
    M, K = x.shape
    flag = torch.zeros(1, dtype=torch.int32, device=x.device)
    y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    check(load().db_decima_linear_w8a32(_ptr(x), M, K, _ptr(w_codes), _ptr(w_scales), N, block, int(fused),
                                        _ptr(bias), _ptr(y), _ptr(flag), _stream()))
    return y


EPILOGUE_STORE, EPILOGUE_RESIDUAL, EPILOGUE_SWIGLU = 0, 1, 2


def tune_gemm(M: int, N: int, K: int, bits: int, epilogue: int = EPILOGUE_STORE, cache_path: str | None = None):
    """Kernel-selection tuner for one GEMM shape (the reference's rule, webgpu/checkpoint.rs:420-565):
    the fastest tile configuration bitwise equal to the default and >= 1 % faster.  Returns
    (GemmConfig, report dict)."""
    import json
    choice = GemmConfig()
    buf = C.create_string_buffer(16384)
    path = cache_path.encode() if cache_path else None
    check(load().db_gemm_tune(M, N, K, bits, epilogue, path, C.byref(choice), buf, len(buf)))
    return choice, json.loads(buf.value.decode())


def linear(x, w_codes, sw, N: int, weight_bits: int = 4, activation_bits: int = 8, fused: bool = True):
    """Matrix::apply (int8.rs:166-176): quantise + grouped GEMM (GEMV path for small M)."""
    import torch
    M, K = x.shape
    ws = torch.empty(load().db_linear_workspace_bytes(M, K), dtype=torch.uint8, device=x.device)
    y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    check(load().db_linear_g64(_ptr(x), M, K, _ptr(w_codes), _ptr(sw), N, weight_bits, activation_bits, int(fused),
                               _ptr(y), _ptr(ws), _stream()))
    return y


def linear_noalloc(x, w_codes, sw, N: int, weight_bits: int = 4, activation_bits: int = 8, fused: bool = True,
                   out=None):
    """Matrix::apply without any device allocation by the library: for hosts that forbid it.  Uses
    the library's fixed scratch array (db_linear_noalloc_scratch_bytes()); see the C header for the
    sharing rules."""
    import torch
    M, K = x.shape
    y = torch.empty((M, N), dtype=torch.float32, device=x.device) if out is None else out
    check(load().db_linear_g64_noalloc(_ptr(x), M, K, _ptr(w_codes), _ptr(sw), N, weight_bits, activation_bits,
                                       int(fused), _ptr(y), _stream()))
    return y


def project_packed(x, w_codes, sw, outputs: int, bits: int):
    """packed::project (packed.rs:75-119) for one activation row."""
    import torch
    K = x.numel()
    ws = torch.empty(load().db_linear_workspace_bytes(1, K), dtype=torch.uint8, device=x.device)
    y = torch.empty(outputs, dtype=torch.float32, device=x.device)
    check(load().db_project_packed(_ptr(x), K, _ptr(w_codes), _ptr(sw), outputs, bits, _ptr(y), _ptr(ws), _stream()))
    return y


def interleave_gate_up(gate_codes, gate_scales, up_codes, up_scales, F: int, K: int, bits: int):
    import torch
    codes = torch.empty((2 * F, gate_codes.shape[1]), dtype=torch.uint8, device=gate_codes.device)
    scales = torch.empty((gate_scales.shape[0], scale_stride(2 * F)), dtype=torch.float32, device=gate_codes.device)
    check(load().db_interleave_gate_up(_ptr(gate_codes), _ptr(gate_scales), _ptr(up_codes), _ptr(up_scales), F, K,
                                       bits, _ptr(codes), _ptr(scales), _stream()))
    return codes, scales


def mlp(a_codes, sa, gu_codes, gu_scales, M: int, F: int, K: int, bits: int, fused: bool = True, nonfinite=None):
    """Fused gate/up + SiLU*up + re-quantisation (grouped_q4_mlp.wgsl) -> (codes [M, F], scales [F/64, M]).
    The code layout follows a_codes: f16 tensor-core codes (db_mlp_g64) or int8 natural codes
    (db_mlp_g64_natural, the kind::i8 path)."""
    import torch
    natural = a_codes.dtype == torch.int8
    codes = torch.zeros((M, F), dtype=torch.int8 if natural else torch.float16, device=a_codes.device)
    scales = torch.zeros((F // GROUP, scale_stride(M)), dtype=torch.float32, device=a_codes.device)
    fn = load().db_mlp_g64_natural if natural else load().db_mlp_g64
    check(fn(_ptr(a_codes), a_codes.stride(0), _ptr(sa), sa.stride(0), _ptr(gu_codes), _ptr(gu_scales),
             M, F, K, bits, int(fused), _ptr(codes), F, _ptr(scales), scale_stride(M), _ptr(nonfinite), _stream()))
    return codes, scales


def attention(q16, k16, v16, q_heads: int, kv_heads: int, scale: float | None = None):
    import torch
    T = q16.shape[0]
    out = torch.empty((T, q_heads * 128), dtype=torch.float32, device=q16.device)
    s = (1.0 / 128 ** 0.5) if scale is None else scale
    check(load().db_attention(_ptr(q16), _ptr(k16), _ptr(v16), T, q_heads, kv_heads, 128, s, _ptr(out),
                              q_heads * 128, _stream()))
    return out


def attention_decoder(q16, k16, v16, items: int, q_heads: int, kv_heads: int, kp16=None, vp16=None,
                      causal: bool = True, scale: float | None = None):
    """Decoder attention: `items` items of q16.shape[0] // items rows, each after the cached prefix
    keys kp16/vp16 [P, kv_heads, 128] (None: no prefix), causal own keys when asked."""
    import torch
    R = q16.shape[0]
    out = torch.empty((R, q_heads * 128), dtype=torch.float32, device=q16.device)
    s = (1.0 / 128 ** 0.5) if scale is None else scale
    P = 0 if kp16 is None else kp16.shape[0]
    check(load().db_attention_decoder(_ptr(q16), _ptr(k16), _ptr(v16), items, R // items,
                                      _ptr(kp16) if P else None, _ptr(vp16) if P else None, P, int(causal), q_heads,
                                      kv_heads, 128, s, _ptr(out), q_heads * 128, _stream()))
    return out


# ------------------------------------------------------------------ generation operators
# A decode step spends microseconds in these wrappers, so their checks read each tensor's shape and
# strides once.
def _heads(name, x, dtype, device: int):
    """A packed tensor [rows, heads, 128] whose rows may be strided (a view of a wider projection) ->
    (rows, heads, row stride)."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != 128:
        raise ValueError(f"{name}: a tensor [rows, heads, 128] is wanted")
    rows, heads, _ = shape
    ld, sh, sd = x.stride()
    if sd != 1 or (sh != 128 and heads > 1):
        raise ValueError(f"{name}: a tensor [rows, heads, 128] with dense rows is wanted")
    if x.dtype != dtype or x.get_device() != device:
        raise ValueError(f"{name}: type or device differs from the other tensors'")
    return rows, heads, ld if rows > 1 else heads * 128


def _array(name, x, dtype, shape, device: int):
    """The address of a dense device tensor of one type and shape; None passes."""
    if x is None:
        return None
    if x.dtype != dtype or x.shape != shape or not x.is_contiguous() or x.get_device() != device:
        raise ValueError(f"{name}: a dense {dtype} tensor {list(shape)} on device {device} is wanted")
    return x.data_ptr()


def _device(name, x) -> int:
    if not x.is_cuda:
        raise ValueError(f"{name}: a tensor on a device is wanted")
    return x.get_device()


def _raw_stream(device: int):
    import torch
    return torch._C._cuda_getCurrentRawStream(device)


# The library launches on the current device, counts its SMs and notes errors in its error word: calls run with the
# tensors' device current.
def _launch(device: int, entry, *args):
    import torch
    if torch._C._cuda_getDevice() == device:
        check(entry(*args, _raw_stream(device)))
    else:
        with torch.cuda.device(device):
            check(entry(*args, _raw_stream(device)))


def _workspace(device: int, like, size, *args):
    """The bytes that size(*args) asks for, from torch's allocator: (tensor, its address), or None twice."""
    import torch
    if torch._C._cuda_getDevice() == device:
        need = size(*args)
    else:
        with torch.cuda.device(device):
            need = size(*args)
    if not need:
        return None, None
    ws = torch.empty(need, dtype=torch.uint8, device=like.device)
    return ws, ws.data_ptr()


def _code16(dtype, name):
    import torch
    if dtype == torch.bfloat16:
        return 2
    if dtype == torch.float16:
        return 1
    raise ValueError(f"{name}: float16 or bfloat16 is wanted")


DELTA_STEP_TOKENS = 16  # DB_DELTA_STEP_TOKENS: up to here items need no workspace


def gated_delta(q, k, v, g, beta, items: int = 1, cu_seqlens=None, max_len: int | None = None, state=None,
                scale: float = 128 ** -0.5, norm_eps: float | None = 1e-6, state_out=None, out=None):
    """The gated delta rule over packed sequences -> (out [rows, v_heads, 128], states after the last rows
    f32 [items, v_heads, 128 (value), 128 (key)]).

    q, k [rows, k_heads, 128], v [rows, v_heads, 128] (f16 or bf16; rows may be views of one wider
    projection), g (log decay) and beta f32 [rows, v_heads].  Without cu_seqlens (int32 [items + 1] on the
    device) the items are equal; with it max_len is the longest item's rows (default: all rows, which
    is only slower).  state: f32 [items, v_heads, 128, 128], or with one item in front a kept state that
    every item starts from; None: zeros.  state_out may be state itself where every
    item has its own, and otherwise shares no memory with it.  q and k are divided by their
    lengths unless norm_eps is None.  A value that is not finite makes the outputs of its value feature (in
    v) or head (elsewhere) NaN, from the start of its block of 64 tokens at the earliest."""
    import torch
    dt, dev = v.dtype, _device("v", v)
    code = _code16(dt, "gated_delta")
    rows, hv, ldv = _heads("v", v, dt, dev)
    rows_k, hk, ldk = _heads("k", k, dt, dev)
    rows_q, hq, ldq = _heads("q", q, dt, dev)
    if rows_k != rows or rows_q != rows or hq != hk:
        raise ValueError("gated_delta: q, k and v differ in their rows or heads")
    f32, ld = torch.float32, []
    for name, x in (("g", g), ("beta", beta)):
        sr, sh = x.stride() if x.dim() == 2 else (0, 0)
        if x.shape != (rows, hv) or x.dtype != f32 or (sh != 1 and hv > 1) or x.get_device() != dev:
            raise ValueError(f"{name}: a float32 tensor [rows, v_heads] with dense rows is wanted")
        ld.append(sr if rows > 1 else hv)
    cu = None
    if cu_seqlens is not None:
        cu = _array("cu_seqlens", cu_seqlens, torch.int32, (items + 1,), dev)
        max_len = rows if max_len is None else min(max_len, rows)
    else:
        if items and rows % items:
            raise ValueError("gated_delta: rows do not divide into equal items")
        max_len = rows // items if items else 0
    stride, si = 0, None
    if state is not None:
        one = len(state.shape) == 4 and state.shape[0] == 1
        si = _array("state", state, f32, (1 if one else items, hv, 128, 128), dev)
        stride = 0 if one and items != 1 else hv * 128 * 128
    if state_out is None:
        state_out = g.new_empty((items, hv, 128, 128))
        so = state_out.data_ptr()
    else:
        so = _array("state_out", state_out, f32, (items, hv, 128, 128), dev)
    if out is None:
        out, ldo = v.new_empty((rows, hv, 128)), hv * 128
    else:
        rows_o, ho, ldo = _heads("out", out, dt, dev)
        if rows_o != rows or ho != hv:
            raise ValueError("gated_delta: out differs from v in its shape")
    lib, ws, at = load(), None, None
    if max_len > DELTA_STEP_TOKENS:
        ws, at = _workspace(dev, v, lib.db_gated_delta_workspace_bytes, items, rows, max_len, hk, hv, code)
    _launch(dev, lib.db_gated_delta, q.data_ptr(), k.data_ptr(), v.data_ptr(), code, ldq, ldk, ldv, g.data_ptr(),
            beta.data_ptr(), ld[0], ld[1], cu, items, rows, max_len, hk, hv, 128, scale,
            -1.0 if norm_eps is None else norm_eps, si, stride, so, out.data_ptr(), ldo, at)
    return out, state_out


class KvCache8:
    """The tensors of an 8-bit paged key/value cache (db_kv8_cache): int8 codes of full blocks of 64 tokens
    with one f32 scale per block, kv head and keys / values, and the open blocks in 16 bits.

    k_codes [pages, kv_heads, 64, 128], v_codes [pages, kv_heads, 128, 64] int8; k_scales, v_scales f32
    [pages, kv_heads]; k_tail [sequences, kv_heads, 64, 128], v_tail [sequences, kv_heads, 128, 64] f16 or
    bf16; page_table int32 [sequences, table_width]: the page of each block, the caller's to fill.  page_table may be set
    to another tensor (a wider one, for longer sequences); the others are fixed, and other tensors another KvCache8."""

    BLOCK = 64
    __slots__ = ("_k_codes", "_k_scales", "_v_codes", "_v_scales", "_k_tail", "_v_tail", "_page_table", "_dtype", "_device",
                 "_kv_heads", "_table_width", "_c", "ref")

    def __init__(self, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, page_table):
        import torch
        dev, dt, f32 = _device("k_tail", k_tail), k_tail.dtype, torch.float32
        if len(k_scales.shape) != 2 or len(page_table.shape) != 2:
            raise ValueError("KvCache8: k_scales [pages, kv_heads] and page_table [sequences, width] are wanted")
        pages, heads = k_scales.shape
        sequences, width = page_table.shape
        code = _code16(dt, "KvCache8")
        c = _lib.KvCache8(
            _array("k_codes", k_codes, torch.int8, (pages, heads, 64, 128), dev),
            _array("k_scales", k_scales, f32, (pages, heads), dev),
            _array("v_codes", v_codes, torch.int8, (pages, heads, 128, 64), dev),
            _array("v_scales", v_scales, f32, (pages, heads), dev),
            _array("k_tail", k_tail, dt, (sequences, heads, 64, 128), dev),
            _array("v_tail", v_tail, dt, (sequences, heads, 128, 64), dev),
            _array("page_table", page_table, torch.int32, (sequences, width), dev),
            pages, width, sequences, heads, 128, code)
        self._k_codes, self._k_scales, self._v_codes, self._v_scales = k_codes, k_scales, v_codes, v_scales
        self._k_tail, self._v_tail, self._page_table = k_tail, v_tail, page_table
        self._dtype, self._device, self._kv_heads, self._table_width = dt, dev, heads, width
        self._c, self.ref = c, C.byref(c)

    # calls read the addresses in _c, so another tensor has to be checked and entered there
    k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, dtype, device, kv_heads, table_width = (
        property(attrgetter("_" + name)) for name in ("k_codes", "k_scales", "v_codes", "v_scales", "k_tail", "v_tail", "dtype",
                                                      "device", "kv_heads", "table_width"))

    @property
    def page_table(self):
        return self._page_table

    @page_table.setter
    def page_table(self, value):
        import torch
        if len(value.shape) != 2:
            raise ValueError("KvCache8: page_table [sequences, width] is wanted")
        width = value.shape[1]
        self._c.page_table = _array("page_table", value, torch.int32, (self._c.sequences, width), self._device)
        self._c.table_width = self._table_width = width
        self._page_table = value

    @classmethod
    def allocate(cls, sequences: int, pages: int, table_width: int, kv_heads: int, dtype, device="cuda") -> "KvCache8":
        """An empty cache; block i of sequence b is page b * table_width + i where the pool is large
        enough for that, else the table is left at -1 (no page) for the caller to fill."""
        import torch
        dev = torch.device(device)
        dev = torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev
        table = torch.full((sequences, table_width), -1, dtype=torch.int32, device=dev)
        if pages >= sequences * table_width:
            table = torch.arange(sequences * table_width, dtype=torch.int32, device=dev).view(sequences, table_width)
        z = lambda dt, *shape: torch.zeros(shape, dtype=dt, device=dev)  # noqa: E731
        return cls(z(torch.int8, pages, kv_heads, 64, 128), z(torch.float32, pages, kv_heads),
                   z(torch.int8, pages, kv_heads, 128, 64), z(torch.float32, pages, kv_heads),
                   z(dtype, sequences, kv_heads, 64, 128), z(dtype, sequences, kv_heads, 128, 64), table)


def _kv8_items(device: int, rows: int, lengths, cu_seqlens, max_rows):
    """(items, their most rows, addresses of lengths and cu_seqlens)."""
    import torch
    if len(lengths.shape) != 1:
        raise ValueError("lengths: a tensor [items] is wanted")
    items = lengths.shape[0]
    ln = _array("lengths", lengths, torch.int32, (items,), device)
    if cu_seqlens is not None:
        cu = _array("cu_seqlens", cu_seqlens, torch.int32, (items + 1,), device)
        return items, rows if max_rows is None else min(max_rows, rows), ln, cu
    if items and rows % items:
        raise ValueError("kv8: rows do not divide into equal items")
    return items, rows // items if items else 0, ln, None


def kv8_append(cache: KvCache8, k, v, lengths, cu_seqlens=None, max_rows: int | None = None) -> None:
    """Writes the items' new rows (k, v [rows, kv_heads, 128]) at positions lengths[b] (int32, device) on;
    blocks that fill up are quantised.  The lengths stay as they are: advance them once every layer has
    taken the step.  cu_seqlens and max_rows as cu_seqlens and max_len in gated_delta, but rows past max_rows or past
    the page table are not cached, and device_error_word notes them."""
    dt, dev = cache._dtype, cache._device
    rows, heads, ldk = _heads("k", k, dt, dev)
    rows_v, heads_v, ldv = _heads("v", v, dt, dev)
    if rows_v != rows or heads_v != heads or heads != cache._kv_heads:
        raise ValueError("kv8_append: k or v differs from the cache in its heads or rows")
    items, most, ln, cu = _kv8_items(dev, rows, lengths, cu_seqlens, max_rows)
    _launch(dev, load().db_kv8_append, cache.ref, k.data_ptr(), ldk, v.data_ptr(), ldv, ln, cu, items, rows, most)


def kv8_attention(cache: KvCache8, q, lengths, cu_seqlens=None, max_rows: int | None = None,
                  max_keys: int | None = None, scale: float = 128 ** -0.5, out=None):
    """Attention over the cache after the append of the same rows: row i of item b sees the cached keys
    0 .. lengths[b] + i -> [rows, q_heads, 128].  max_keys: the longest item's keys, as far as the caller
    knows (default: the table's width); it only sizes the launch and the workspace.  Rows that the append left out
    are 0."""
    dt, dev = cache._dtype, cache._device
    rows, heads, ldq = _heads("q", q, dt, dev)
    items, most, ln, cu = _kv8_items(dev, rows, lengths, cu_seqlens, max_rows)
    if out is None:
        out, ldo = q.new_empty((rows, heads, 128)), heads * 128
    else:
        rows_o, heads_o, ldo = _heads("out", out, dt, dev)
        if rows_o != rows or heads_o != heads:
            raise ValueError("kv8_attention: out differs from q in its shape")
    lib, keys = load(), max(1, max_keys or cache._table_width * 64)
    ws, at = _workspace(dev, q, lib.db_kv8_attention_workspace_bytes, items, most, keys, cache._kv_heads, heads)
    _launch(dev, lib.db_kv8_attention, cache.ref, q.data_ptr(), ldq, ln, cu, items, rows, most, keys, heads, scale,
            out.data_ptr(), ldo, at)
    return out


def kv8_read(cache: KvCache8, lengths, max_keys: int):
    """The cached keys and values of tokens 0 .. max_keys - 1, f32 [items, max_keys, kv_heads, 128] each
    (0 from lengths[b] on)."""
    import torch
    dev = cache._device
    items, _, ln, _ = _kv8_items(dev, 0, lengths, None, None)
    k, v = (torch.empty((items, max_keys, cache._kv_heads, 128), dtype=torch.float32, device=cache._k_tail.device)
            for _ in range(2))
    _launch(dev, load().db_kv8_read, cache.ref, ln, items, max_keys, k.data_ptr(), v.data_ptr())
    return k, v


def logit_rules(logits, history=None, history_lengths=None, repetition=None, presence=None, frequency=None,
                bias_ids=None, bias_values=None, mask=None, out=None):
    """Penalties for repeated tokens, biases and a grammar mask on logits [rows, vocab] -> (values f32
    [rows, vocab], best token int32 [rows], log-sum-exp f32 [rows]); values - lse are log-probabilities.

    history int32 [rows, n] with history_lengths int32 [rows] (None: all n); repetition, presence and
    frequency f32 [rows]; bias_ids int32 and bias_values f32 [rows, m]; mask int32 [rows, ceil(vocab / 32)],
    bit id % 32 of word id / 32 set where a token is allowed.  A row with nothing allowed has best -1
    and lse -inf.  out may be f32 logits themselves."""
    import torch
    f32, i32, dt = torch.float32, torch.int32, logits.dtype
    if len(logits.shape) != 2:
        raise ValueError("logit_rules: logits [rows, vocab] are wanted")
    rows, vocab = logits.shape
    ld, step = logits.stride()
    dev = _device("logits", logits)
    if vocab > 1 and step != 1:
        raise ValueError("logit_rules: logits with dense rows are wanted")
    if dt != f32 and dt != torch.float16 and dt != torch.bfloat16:
        raise ValueError("logit_rules: logits are float32, float16 or bfloat16")
    cols = history.shape[1] if history is not None else 0
    biases = bias_ids.shape[1] if bias_ids is not None else 0
    words, one = (vocab + 31) // 32, (rows,)
    if out is None:
        out, ldo = torch.empty((rows, vocab), dtype=f32, device=logits.device), vocab
    else:
        ldo, step = out.stride() if len(out.shape) == 2 else (0, 0)
        if out.shape != logits.shape or out.dtype != f32 or (vocab > 1 and step != 1) or out.get_device() != dev:
            raise ValueError("logit_rules: out is f32 with dense rows, of the logits' shape")
    best, lse = out.new_empty(one, dtype=i32), out.new_empty(one)
    _launch(
        dev, load().db_logit_rules,
        logits.data_ptr(), 0 if dt == f32 else 1 if dt == torch.float16 else 2, ld if rows > 1 else vocab, rows, vocab,
        _array("history", history, i32, (rows, cols), dev), cols,
        _array("history_lengths", history_lengths, i32, one, dev), cols, _array("repetition", repetition, f32, one, dev),
        _array("presence", presence, f32, one, dev), _array("frequency", frequency, f32, one, dev),
        _array("bias_ids", bias_ids, i32, (rows, biases), dev),
        _array("bias_values", bias_values, f32, (rows, biases), dev), biases, _array("mask", mask, i32, (rows, words), dev),
        words, out.data_ptr(), ldo if rows > 1 else vocab, best.data_ptr(), lse.data_ptr())
    return out, best, lse


def synthetic_bf16(seed: int, tensor: int, shape, std: float, device="cuda"):
    import torch
    out = torch.empty(shape, dtype=torch.int16, device=device)
    check(load().db_synthetic_bf16(seed, tensor, out.numel(), std, _ptr(out), _stream()))
    return out


def device_error_word() -> int:
    return int(load().db_device_error_word())


# ------------------------------------------------------------------ model level (inference API mirror)
class Error(Exception):
    """inference::Error {code, message} (src/inference/mod.rs:44-85)."""

    def __init__(self, code: str, message: str):
        super().__init__(f"{code}: {message}")
        self.code, self.message = code, message

    @staticmethod
    def _from(e: _lib.DbError) -> "Error":
        return Error(e.code.decode(), e.message.decode())


class Cancellation:
    """inference::Cancellation (mod.rs:87-100): a shared flag the library polls."""

    def __init__(self):
        self._flag = C.c_uint8(0)  # the layout of Rust's AtomicBool

    def cancel(self):
        self._flag.value = 1

    def check(self):
        if self._flag.value:
            raise Error("CANCELLED", "Inference was cancelled")

    @property
    def ptr(self):
        return C.byref(self._flag)


@dataclass
class CacheOptions:
    """inference::CacheOptions (mod.rs:102-115)."""
    max_bytes: int = 64 * 1024 * 1024
    require_prefix: bool = False


@dataclass
class PplxParameters:
    """inference::PplxParameters (parameters.rs:81-103)."""
    max_sequence_tokens: int = 1024


@dataclass
class EncoderConfig:
    layers: int = 28
    hidden: int = 1024
    q_heads: int = 16
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 3072
    vocab: int = 151936
    weight_bits: int = 4
    rope_theta: float = 1e6
    eps: float = 1e-6
    max_sequence_tokens: int = 1024
    fused: bool = True
    causal: bool = False  # True: decoder (causal attention, prefix caches)

    def c(self) -> _lib.EncoderConfig:
        return _lib.EncoderConfig(self.layers, self.hidden, self.q_heads, self.kv_heads, self.head_dim, self.ffn,
                                  self.vocab, self.weight_bits, self.rope_theta, self.eps, self.max_sequence_tokens,
                                  int(self.fused), int(self.causal))


@dataclass
class Response:
    """inference::Response (mod.rs:127-132); `response` is the pooled embedding."""
    response: object
    model: str
    backend: str


@dataclass
class Outcome:
    """inference::Outcome (mod.rs:133-138)."""
    status: str
    result: Response | None = None
    error: Error | None = None


class Cache:
    def __init__(self, handle, model):
        self._h, self._model = handle, model

    def stats(self) -> dict:
        """Prefix reuse counters (kev/mod.rs Stats): hits, prefix tokens reused / computed."""
        v = (C.c_int64 * 3)()
        check(load().db_cache_stats(self._h, C.byref(v, 0), C.byref(v, 8), C.byref(v, 16)))
        return {"hits": v[0], "prefix_tokens_reused": v[1], "prefix_tokens_computed": v[2]}

    def __del__(self):
        if getattr(self, "_h", None):
            load().db_cache_destroy(self._h)
            self._h = None


class Model:
    """inference::Model<B> (mod.rs:156-273) over the CUDA encoder backend."""

    def __init__(self, handle, config: EncoderConfig):
        self._h, self.config = handle, config
        self.defaults = PplxParameters(config.max_sequence_tokens)

    @classmethod
    def synthetic(cls, config: EncoderConfig, seed: int = 0, std: float = 0.02, device: int = 0) -> "Model":
        err = _lib.DbError()
        cfg = config.c()
        h = load().db_model_create_synthetic(device, C.byref(cfg), seed, std, C.byref(err))
        if not h:
            raise Error._from(err)
        return cls(h, config)

    @classmethod
    def from_weights(cls, config: EncoderConfig, weights: dict, device: int = 0) -> "Model":
        """weights: 'embedding' bf16 bits [vocab, hidden]; per-layer lists 'q','k','v','o','gate','up','down'
        (bf16 bits [out, in]); per-layer f32 'input_norm','post_norm','q_norm','k_norm'; 'final_norm'."""
        import numpy as np
        keep = []

        def arr(a, dt):
            a = np.ascontiguousarray(a, dtype=dt)
            keep.append(a)
            return a.ctypes.data_as(C.POINTER(C.c_uint16 if dt == np.uint16 else C.c_float))

        w = _lib.EncoderWeights()
        w.embedding = arr(weights["embedding"], np.uint16)
        L = config.layers
        for n in ("q", "k", "v", "o", "gate", "up", "down"):
            p = (C.POINTER(C.c_uint16) * L)(*[arr(t, np.uint16) for t in weights[n]])
            keep.append(p)
            setattr(w, n, C.cast(p, _lib._u16pp))
        for n in ("input_norm", "post_norm", "q_norm", "k_norm"):
            p = (C.POINTER(C.c_float) * L)(*[arr(t, np.float32) for t in weights[n]])
            keep.append(p)
            setattr(w, n, C.cast(p, _lib._fpp))
        w.final_norm = arr(weights["final_norm"], np.float32)
        err = _lib.DbError()
        cfg = config.c()
        h = load().db_model_create(device, C.byref(cfg), C.byref(w), C.byref(err))
        if not h:
            raise Error._from(err)
        return cls(h, config)

    def close(self):
        if getattr(self, "_h", None):
            load().db_model_destroy(self._h)
            self._h = None

    __del__ = close

    def capabilities(self) -> dict:
        buf = C.create_string_buffer(512)
        check(load().db_model_capabilities(self._h, buf, 512))
        return json.loads(buf.value.decode())

    def synthetic_weight(self, name: str, layer: int = 0):
        import numpy as np
        n = load().db_model_synthetic_weight(self._h, name.encode(), layer, None, 0)
        if n < 0:
            raise CudaError(int(n))
        out = np.empty(n, dtype=np.uint16)
        got = load().db_model_synthetic_weight(self._h, name.encode(), layer, out.ctypes.data_as(C.c_void_p), n)
        if got != n:
            raise CudaError(int(got))
        return out

    def create_cache(self, options: CacheOptions | None = None) -> Cache:
        o = options or CacheOptions()
        err = _lib.DbError()
        h = load().db_cache_create(self._h, o.max_bytes, int(o.require_prefix), C.byref(err))
        if not h:
            raise Error._from(err)
        return Cache(h, self)

    def clear_cache(self, cache: Cache):
        err = _lib.DbError()
        if load().db_cache_clear(self._h, cache._h, C.byref(err)):
            raise Error._from(err)

    def _params(self, parameters):
        p = parameters or self.defaults
        return _lib.Parameters(p.max_sequence_tokens)

    def predict(self, ids, parameters: PplxParameters | None = None, cache: Cache | None = None,
                cancellation: Cancellation | None = None, out=None) -> Response:
        import numpy as np
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        out = np.empty(self.config.hidden, dtype=np.float32) if out is None else out
        err = _lib.DbError()
        p = self._params(parameters)
        rc = load().db_predict(self._h, ids.ctypes.data_as(C.c_void_p), ids.size, C.byref(p),
                               cache._h if cache else None, cancellation.ptr if cancellation else None,
                               out.ctypes.data_as(C.c_void_p), C.byref(err))
        if rc:
            raise Error._from(err)
        caps = self.capabilities()
        return Response(out, caps["model"], caps["backend"])

    def predict_continuations(self, prefix, continuations, cache: Cache | None = None,
                              cancellation: Cancellation | None = None):
        """Causal models: the final-normed hidden states [count, tokens, hidden] of each continuation
        (equal-length token lists) after a shared prefix, whose per-layer keys and values are
        computed once or reused from the cache (kev/mod.rs:163-300)."""
        import numpy as np
        pre = np.ascontiguousarray(prefix, dtype=np.int32)
        cont = np.ascontiguousarray(continuations, dtype=np.int32)
        if cont.ndim != 2:
            raise ValueError("continuations must be equal-length token lists")
        out = np.empty((cont.shape[0], cont.shape[1], self.config.hidden), dtype=np.float32)
        err = _lib.DbError()
        rc = load().db_predict_continuations(self._h, cache._h if cache else None, pre.ctypes.data_as(C.c_void_p),
                                             pre.size, cont.ctypes.data_as(C.c_void_p), cont.shape[0], cont.shape[1],
                                             cancellation.ptr if cancellation else None,
                                             out.ctypes.data_as(C.c_void_p), C.byref(err))
        if rc:
            raise Error._from(err)
        return out

    def score_continuations(self, prefix, continuations, cache: Cache | None = None,
                            cancellation: Cancellation | None = None, hidden: bool = False):
        """Causal models: per-token log-probabilities [count, tokens] of each continuation after the
        shared prefix, from an LM head tied to the embedding matrix (the continuation's score is
        the row sum).  With hidden=True also the LM head's input rows [1 + count*tokens, hidden]:
        the prefix's last final-normed state, then the continuations' states."""
        import numpy as np
        pre = np.ascontiguousarray(prefix, dtype=np.int32)
        cont = np.ascontiguousarray(continuations, dtype=np.int32)
        if cont.ndim != 2:
            raise ValueError("continuations must be equal-length token lists")
        out = np.empty(cont.shape, dtype=np.float32)
        h = np.empty((1 + cont.size, self.config.hidden), dtype=np.float32) if hidden else None
        err = _lib.DbError()
        rc = load().db_score_continuations(self._h, cache._h if cache else None, pre.ctypes.data_as(C.c_void_p),
                                           pre.size, cont.ctypes.data_as(C.c_void_p), cont.shape[0], cont.shape[1],
                                           cancellation.ptr if cancellation else None,
                                           out.ctypes.data_as(C.c_void_p),
                                           h.ctypes.data_as(C.c_void_p) if h is not None else None, C.byref(err))
        if rc:
            raise Error._from(err)
        return (out, h) if hidden else out

    def predict_batch(self, requests, parameters: PplxParameters | None = None, cache: Cache | None = None,
                      cancellation: Cancellation | None = None) -> list[Outcome]:
        import numpy as np
        reqs = [np.ascontiguousarray(r, dtype=np.int32) for r in requests]
        n = len(reqs)
        ptrs = (C.c_void_p * max(n, 1))(*[r.ctypes.data_as(C.c_void_p).value for r in reqs])
        lens = (C.c_size_t * max(n, 1))(*[r.size for r in reqs])
        outs = np.zeros((max(n, 1), self.config.hidden), dtype=np.float32)
        status = np.zeros(max(n, 1), dtype=np.int32)
        errs = (_lib.DbError * max(n, 1))()
        err = _lib.DbError()
        p = self._params(parameters)
        rc = load().db_predict_batch(self._h, ptrs, lens, n, C.byref(p), cache._h if cache else None,
                                     cancellation.ptr if cancellation else None, outs.ctypes.data_as(C.c_void_p),
                                     status.ctypes.data_as(C.c_void_p), errs, C.byref(err))
        if rc:
            raise Error._from(err)
        caps = self.capabilities()
        result = []
        for i in range(n):
            if status[i] == 0:
                result.append(Outcome("success", result=Response(outs[i].copy(), caps["model"], caps["backend"])))
            else:
                result.append(Outcome("error", error=Error._from(errs[i])))
        return result

    def use_graphs(self, enable: bool = True):
        """Forward as a captured CUDA graph per token count (default on); bit-identical either way."""
        check(load().db_model_use_graphs(self._h, int(enable)))

    def set_code_layout(self, layout: int):
        """CODES_NATURAL (int8 codes, kind::i8 GEMM; default) or CODES_TC (f16 codes, kind::f16 GEMM),
        bit-identical outputs either way; or CODES_DQ (dequantised f16 operands, full-K f32
        accumulation: within the contract's tolerance, not bit-identical)."""
        check(load().db_model_set_code_layout(self._h, int(layout)))

    def profile(self, enable: bool = True):
        check(load().db_model_profile(self._h, int(enable)))

    def profile_read(self, reset: bool = True) -> dict:
        """{kernel kind: (total ms, launches)} accumulated since the last reset."""
        import numpy as np
        n = 11
        ms = np.zeros(n, np.float64)
        cnt = np.zeros(n, np.int64)
        check(load().db_model_profile_read(self._h, ms.ctypes.data_as(C.c_void_p), cnt.ctypes.data_as(C.c_void_p), n,
                                           int(reset)))
        return {load().db_model_profile_name(k).decode(): (float(ms[k]), int(cnt[k])) for k in range(n)}

    @classmethod
    def from_packed(cls, config: EncoderConfig, manifest_path: str, verify: bool = True, device: int = 0) -> "Model":
        """Loads a packed checkpoint directory (packed-q4-e4.json / packed-q8-e8.json manifest, the
        reference's export_packed.rs format); verify checks every file's SHA-256."""
        err = _lib.DbError()
        cfg = config.c()
        h = load().db_model_create_packed(device, C.byref(cfg), manifest_path.encode(), int(verify), C.byref(err))
        if not h:
            raise Error._from(err)
        return cls(h, config)

    def set_streaming(self, enable: bool = True):
        """Two-bank layer streaming: weights in pinned host memory, two layers on the device."""
        err = _lib.DbError()
        if load().db_model_set_streaming(self._h, int(enable), C.byref(err)):
            raise Error._from(err)

    def export_packed(self, directory: str) -> str:
        """Writes this model's weights as a packed checkpoint into directory; returns the manifest path."""
        import os
        err = _lib.DbError()
        if load().db_model_export_packed(self._h, directory.encode(), C.byref(err)):
            raise Error._from(err)
        return os.path.join(directory, f"packed-q{self.config.weight_bits}-e{self.config.weight_bits}.json")

    def tune(self, tokens: int | None = None, cache_path: str | None = None) -> dict:
        """Tunes the four projection GEMMs at `tokens` rows (default: max_sequence_tokens) and uses
        the choices from then on; returns the per-projection reports."""
        import json
        err = _lib.DbError()
        buf = C.create_string_buffer(65536)
        n = tokens if tokens is not None else self.config.max_sequence_tokens
        rc = load().db_model_tune(self._h, n, cache_path.encode() if cache_path else None, buf, len(buf), C.byref(err))
        if rc:
            raise Error._from(err)
        return json.loads(buf.value.decode())

    def forward_device(self, ids_dev, out_dev, stream=None):
        """Device-resident forward (no host synchronisation) used for device-timed measurement."""
        check(load().db_forward_device(self._h, _ptr(ids_dev), ids_dev.numel(), _ptr(out_dev), _stream(stream)))


@dataclass
class BertConfig:
    """C4: the Decima-shaped (BERT) encoder on the Decima int8 kernels (db_bert_*)."""
    layers: int = 12
    hidden: int = 768
    heads: int = 12
    ffn: int = 3072
    vocab: int = 128100
    max_positions: int = 512
    block: int = 32
    eps: float = 1e-12
    fused: bool = True
    mode: int = 0  # 0: W8A8 (WeightsActivations), 1: W8A32 (Weights)

    def c(self) -> _lib.BertConfig:
        return _lib.BertConfig(self.layers, self.hidden, self.heads, self.ffn, self.vocab, self.max_positions,
                               self.block, self.eps, int(self.fused), int(self.mode))


class BertModel:
    """Synthetic-weight C4 encoder; predict returns (mean-pooled [hidden], states [n, hidden])."""

    def __init__(self, config: BertConfig, seed: int = 0, std: float = 0.02, device: int = 0):
        err = _lib.DbError()
        cfg = config.c()
        self._h = load().db_bert_create_synthetic(device, C.byref(cfg), seed, std, C.byref(err))
        if not self._h:
            raise Error._from(err)
        self.config, self.seed, self.std = config, seed, std

    def predict(self, ids, hidden: bool = False):
        import numpy as np
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        pooled = np.empty(self.config.hidden, np.float32)
        h = np.empty((ids.size, self.config.hidden), np.float32) if hidden else None
        err = _lib.DbError()
        rc = load().db_bert_predict(self._h, ids.ctypes.data_as(C.c_void_p), ids.size,
                                    pooled.ctypes.data_as(C.c_void_p),
                                    h.ctypes.data_as(C.c_void_p) if h is not None else None, C.byref(err))
        if rc:
            raise Error._from(err)
        return (pooled, h) if hidden else pooled

    HEAD_OUTPUTS = 3

    def score(self, state, choices, pooled: bool = False):
        """One cross-encoder request: logits [len(choices), 3] for the sequences state ++ choice,
        run packed in one pass (and their pooled states [len(choices), hidden] when asked)."""
        import numpy as np
        state = np.ascontiguousarray(state, dtype=np.int32)
        chs = [np.ascontiguousarray(c, dtype=np.int32) for c in choices]
        ptrs = (C.c_void_p * max(len(chs), 1))(*[c.ctypes.data for c in chs])
        lens = (C.c_size_t * max(len(chs), 1))(*[c.size for c in chs])
        logits = np.empty((len(chs), self.HEAD_OUTPUTS), np.float32)
        p = np.empty((len(chs), self.config.hidden), np.float32) if pooled else None
        err = _lib.DbError()
        rc = load().db_bert_score(self._h, state.ctypes.data_as(C.c_void_p), state.size, ptrs, lens, len(chs),
                                  logits.ctypes.data_as(C.c_void_p),
                                  p.ctypes.data_as(C.c_void_p) if p is not None else None, C.byref(err))
        if rc:
            raise Error._from(err)
        return (logits, p) if pooled else logits

    def close(self):
        if getattr(self, "_h", None):
            load().db_bert_destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()
