"""torch-facing wrappers over the C ABI (device tensors in, device tensors out).

Each function validates shapes on the host, passes raw device pointers and the
current HIP stream to the corresponding ``kdq_*`` entry point, and raises
``KdqError`` on a non-zero status.  Nothing here computes on the CPU.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import BLOCK_BYTES, BLOCK_VALUES, MatvecJob, call, lib


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # (not a public name)
# (the same, without a check that the device runtime is up, which a device tensor stands for)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream() -> int:
    """The current HIP stream.  A decode product takes 6-8 us on the device, so its wrapper must
    not take longer: the raw handle, where torch gives it, without the Stream object
    torch.cuda.current_stream() builds."""
    if _raw_stream is None or not torch.cuda.is_initialized():
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, n_in]."""
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def _need(t: torch.Tensor, dtype, name: str) -> None:
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} device tensor")


def dequantize(encoding: int, packed: torch.Tensor, n_in: int,
               status: torch.Tensor | None = None) -> torch.Tensor:
    """packed: uint8 [rows, row_bytes] -> fp32 [rows, n_in] (kdq_dequantize)."""
    _need(packed, torch.uint8, "packed")
    rows = packed.shape[0]
    out = torch.empty(rows, n_in, dtype=torch.float32, device=packed.device)
    call("kdq_dequantize", encoding, packed.data_ptr(), packed.shape[1], rows, n_in,
         out.data_ptr(), _ptr(status), _stream())
    return out


def gemv(encoding: int, weights: torch.Tensor, x: torch.Tensor, n_out: int,
         out: torch.Tensor | None = None, status: torch.Tensor | None = None,
         exact: bool = False) -> torch.Tensor:
    """y[r, c] = sum_k decode(W[c, k]) x[r, k].  weights uint8 [n_out, row_bytes],
    x fp32 [rows, n_in] -> y fp32 [rows, n_out] (kdq_gemv / kdq_gemv_exact)."""
    _need(weights, torch.uint8, "weights")
    _need(x, torch.float32, "x")
    x2 = _rows(x)
    rows, n_in = x2.shape
    if weights.shape[0] != n_out:
        raise ValueError("weights rows != n_out")
    if out is None:
        out = torch.empty(rows, n_out, dtype=torch.float32, device=x.device)
    fn = "kdq_gemv_exact" if exact else "kdq_gemv"
    call(fn, encoding, weights.data_ptr(), weights.shape[1], x2.data_ptr(), rows, n_in, n_out,
         out.data_ptr(), out.stride(0) if out.dim() == 2 else n_out, _ptr(status), _stream())
    return out


def gemv_batch(jobs: list[dict]) -> None:
    """One submission of several products (kdq_gemv_batch).  Each job: dict with
    encoding, weights (uint8 [columns, row_bytes]), input (fp32 [rows, in]),
    output (fp32 [rows, stride]), optional status."""
    import ctypes as C
    table = (MatvecJob * len(jobs))()
    for i, j in enumerate(jobs):
        w, x, y = j["weights"], j["input"], j["output"]
        x2 = _rows(x)
        table[i] = MatvecJob(w.data_ptr(), x2.data_ptr(), y.data_ptr(),
                             _ptr(j.get("status")) or 0, w.shape[1],
                             y.stride(0) if y.dim() == 2 else w.shape[0],
                             x2.shape[1], w.shape[0], x2.shape[0], j["encoding"])
    call("kdq_gemv_batch", C.addressof(table) if jobs else None, len(jobs), _stream())


@functools.lru_cache(maxsize=4096, typed=True)  # (256.0 is refused, also after 256)
def _packed_bytes(encoding: int, n_in: int, n_out: int) -> int:
    return int(lib().kdq_gguf_packed_bytes(encoding, n_in, n_out))


def gguf_packed_bytes(encoding: int, n_in: int, n_out: int) -> int:
    lib()  # (raises where the library is missing, also for a size asked before)
    return _packed_bytes(encoding, n_in, n_out)


def gguf_pack(encoding: int, weights: torch.Tensor, n_in: int) -> torch.Tensor:
    """Row-major packed rows uint8 [n_out, row_bytes] -> the tile-packed resident form,
    uint8 [kdq_gguf_packed_bytes] (kdq_gguf_pack)."""
    _need(weights, torch.uint8, "weights")
    n_out = weights.shape[0]
    nbytes = gguf_packed_bytes(encoding, n_in, n_out)
    if not nbytes:
        raise ValueError("shape has no packed form (in % 256 != 0)")
    out = torch.empty(nbytes, dtype=torch.uint8, device=weights.device)
    call("kdq_gguf_pack", encoding, weights.data_ptr(), weights.shape[1], n_in, n_out,
         out.data_ptr(), _stream())
    return out


def gemv_packed(encoding: int, packed: torch.Tensor, x: torch.Tensor, n_out: int,
                out: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """gemv over tile-packed weights (kdq_gemv_packed)."""
    _need(packed, torch.uint8, "packed")
    _need(x, torch.float32, "x")
    x2 = _rows(x)
    rows, n_in = x2.shape
    if packed.numel() != _packed_bytes(encoding, n_in, n_out):
        raise ValueError("packed size does not match (encoding, n_in, n_out)")
    if out is None:
        out = torch.empty(rows, n_out, dtype=torch.float32, device=x.device)
    call("kdq_gemv_packed", encoding, packed.data_ptr(), x2.data_ptr(), rows, n_in, n_out,
         out.data_ptr(), out.stride(0) if out.dim() == 2 else n_out, _ptr(status), _stream())
    return out


def gemv_packed_batch(jobs: list[dict]) -> None:
    """One submission over packed weights (kdq_gemv_packed_batch).  Each job: dict with
    encoding, weights (packed uint8), columns, input (fp32 [rows, in]), output
    (fp32 [rows, stride]), optional status."""
    import ctypes as C
    table = (MatvecJob * len(jobs))()
    for i, j in enumerate(jobs):
        w, x, y = j["weights"], j["input"], j["output"]
        x2 = _rows(x)
        table[i] = MatvecJob(w.data_ptr(), x2.data_ptr(), y.data_ptr(),
                             _ptr(j.get("status")) or 0, 0,
                             y.stride(0) if y.dim() == 2 else j["columns"],
                             x2.shape[1], j["columns"], x2.shape[0], j["encoding"])
    call("kdq_gemv_packed_batch", C.addressof(table) if jobs else None, len(jobs), _stream())


def quantize_q8(x_f16: torch.Tensor):
    """fp16 [m, k] -> (int8 [m, k], fp32 [m, k/32]) (kdq_quantize_q8)."""
    _need(x_f16, torch.float16, "x")
    m, k = x_f16.shape
    q = torch.empty(m, k, dtype=torch.int8, device=x_f16.device)
    d = torch.empty(m, k // 32, dtype=torch.float32, device=x_f16.device)
    call("kdq_quantize_q8", x_f16.data_ptr(), m, k, q.data_ptr(), d.data_ptr(), _stream())
    return q, d


def gemm_q4_0(weights: torch.Tensor, x_f16: torch.Tensor, n_out: int,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Q4_0 weights uint8 [n_out, k/32*18] x fp16 [m, k] -> fp16 [m, n_out] (kdq_gemm_q4_0)."""
    _need(weights, torch.uint8, "weights")
    _need(x_f16, torch.float16, "x")
    m, k = x_f16.shape
    if out is None:
        out = torch.empty(m, n_out, dtype=torch.float16, device=x_f16.device)
    call("kdq_gemm_q4_0", weights.data_ptr(), n_out, k, x_f16.data_ptr(), m, out.data_ptr(),
         _stream())
    return out


def gemm_q4_0_packed(packed: torch.Tensor, x_f16: torch.Tensor, n_out: int,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Tile-packed Q4_0 weights (gguf_pack) x fp16 [m, k] -> fp16 [m, n_out]
    (kdq_gemm_q4_0_packed)."""
    _need(packed, torch.uint8, "packed")
    _need(x_f16, torch.float16, "x")
    m, k = x_f16.shape
    if packed.numel() != _packed_bytes(2, k, n_out):  # KDQ_Q4_0
        raise ValueError("packed size does not match (k, n_out)")
    if out is None:
        out = torch.empty(m, n_out, dtype=torch.float16, device=x_f16.device)
    call("kdq_gemm_q4_0_packed", packed.data_ptr(), n_out, k, x_f16.data_ptr(), m,
         out.data_ptr(), _stream())
    return out


def gemm_packed(encoding: int, packed: torch.Tensor, x: torch.Tensor, n_out: int,
                out: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """Tile-packed Q4_K / Q8_0 / Q6_K weights (gguf_pack) x fp32 [m, k] -> fp32 [m, n_out]
    (kdq_gemm_packed, the prefill product)."""
    _need(packed, torch.uint8, "packed")
    _need(x, torch.float32, "x")
    m, k = x.shape
    if packed.numel() != _packed_bytes(encoding, k, n_out):
        raise ValueError("packed size does not match (k, n_out)")
    if out is None:
        out = torch.empty(m, n_out, dtype=torch.float32, device=x.device)
    call("kdq_gemm_packed", encoding, packed.data_ptr(), n_out, k, x.data_ptr(), m,
         out.data_ptr(), _ptr(status), _stream())
    return out


def gemm_rows(encoding: int, w: torch.Tensor, x: torch.Tensor, n_out: int,
              out: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """Row-major GGUF rows [n_out, row_bytes] (uint8, as the file holds them) x fp32
    [m, k] -> fp32 [m, n_out] (kdq_gemm_rows, the prefill product of every encoding)."""
    _need(w, torch.uint8, "w")
    _need(x, torch.float32, "x")
    m, k = x.shape
    if w.dim() != 2 or w.shape[0] != n_out:
        raise ValueError("w must be [n_out, row_bytes]")
    if out is None:
        out = torch.empty(m, n_out, dtype=torch.float32, device=x.device)
    call("kdq_gemm_rows", encoding, w.data_ptr(), w.shape[1], n_out, k, x.data_ptr(), m,
         out.data_ptr(), _ptr(status), _stream())
    return out


def gguf_gemm_check(encoding: int, packed: torch.Tensor, n_out: int, n_in: int) -> int:
    """The prefill GEMM's scale checks over a tile-packed matrix (kdq_gguf_gemm_check):
    bit 1 a non-finite scale, bit 2 a dequantised weight that could pass the fp16 range
    (waits for the device)."""
    flags = torch.zeros(1, dtype=torch.int32, device=packed.device)
    call("kdq_gguf_gemm_check", encoding, packed.data_ptr(), n_out, n_in, flags.data_ptr(),
         _stream())
    return int(flags.item())


def moe_gguf_pack(spec: dict) -> dict:
    """Tile-packed copies (kdq_gguf_pack) of a GGUF MoE spec's expert stacks and shared
    matrices, for moe_gguf(..., packed=...): name -> uint8 device tensor, for the
    encodings the prefill GEMM reads packed (Q4_K, Q8_0, Q6_K), and "checked": every copy
    passed kdq_gguf_gemm_check with no flag."""
    from . import MOE_GGUF_TENSORS
    H, F, S = spec["hidden"], spec["ff"], spec["shared_ff"]
    shape = {"gate_exps": (H, F), "up_exps": (H, F), "down_exps": (F, H),
             "gate_shexp": (H, S), "up_shexp": (H, S), "down_shexp": (S, H)}
    out = {}
    for name in MOE_GGUF_TENSORS[1:]:
        enc, t = spec[name]
        if enc not in (12, 8, 14):  # Q4_K, Q8_0, Q6_K
            continue
        n_in, rows = shape[name]
        count = rows * (t.shape[0] if t.dim() == 3 else 1)
        out[name] = gguf_pack(enc, t.reshape(count, t.shape[-1]), n_in)
    out["checked"] = all(gguf_gemm_check(spec[n][0], out[n], shape[n][1] * (
        spec[n][1].shape[0] if spec[n][1].dim() == 3 else 1), shape[n][0]) == 0
        for n in list(out))
    return out


def moe_gguf(spec: dict, x: torch.Tensor, status: torch.Tensor | None = None,
             packed: dict | None = None):
    """GGUF MoE layer (kdq_moe_gguf; kdq_moe_gguf_packed when `packed` holds resident
    tile-packed copies from moe_gguf_pack).  spec: hidden, experts, top_k, ff, shared_ff,
    shared_gate (fp32 device tensor [hidden]) and per tensor name (encoding, uint8 device
    tensor [rows, row_bytes] or [experts, rows, row_bytes]).  x fp32 [rows, hidden] ->
    (y fp32 [rows, hidden], selected int32 [rows, top_k], weights fp32 [rows, top_k])."""
    from . import MOE_GGUF_TENSORS, GgufTensor, MoeGgufLayer, MoeGgufPackedStacks
    _need(x, torch.float32, "x")
    layer = MoeGgufLayer(spec["hidden"], spec["experts"], spec["top_k"], spec["ff"],
                         spec["shared_ff"])
    for name in MOE_GGUF_TENSORS:
        enc, t = spec[name]
        _need(t, torch.uint8, name)
        expert_bytes = t.shape[1] * t.shape[2] if t.dim() == 3 else 0
        setattr(layer, name, GgufTensor(t.data_ptr(), t.shape[-1], expert_bytes, enc))
    _need(spec["shared_gate"], torch.float32, "shared_gate")
    layer.shared_gate = spec["shared_gate"].data_ptr()
    rows = x.shape[0]
    y = torch.empty(rows, spec["hidden"], dtype=torch.float32, device=x.device)
    sel = torch.empty(rows, spec["top_k"], dtype=torch.int32, device=x.device)
    w = torch.empty(rows, spec["top_k"], dtype=torch.float32, device=x.device)
    if packed is None:
        call("kdq_moe_gguf", ctypes.addressof(layer), x.data_ptr(), rows, y.data_ptr(),
             sel.data_ptr(), w.data_ptr(), _ptr(status), _stream())
    else:
        stacks = MoeGgufPackedStacks(*[packed[n].data_ptr() if n in packed else None
                                       for n in MOE_GGUF_TENSORS[1:]],
                                     int(bool(packed.get("checked", False))))
        call("kdq_moe_gguf_packed", ctypes.addressof(layer), ctypes.addressof(stacks),
             x.data_ptr(), rows, y.data_ptr(), sel.data_ptr(), w.data_ptr(), _ptr(status),
             _stream())
    return y, sel, w


def moe_route(logits: torch.Tensor, top_k: int):
    """fp32 [tokens, experts] -> idx, w, offsets, perm (kdq_moe_route)."""
    _need(logits, torch.float32, "logits")
    t, e = logits.shape
    dev = logits.device
    idx = torch.empty(t, top_k, dtype=torch.int32, device=dev)
    w = torch.empty(t, top_k, dtype=torch.float32, device=dev)
    offsets = torch.empty(e + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(t * top_k, dtype=torch.int32, device=dev)
    call("kdq_moe_route", logits.data_ptr(), t, e, top_k, idx.data_ptr(), w.data_ptr(),
         offsets.data_ptr(), perm.data_ptr(), _stream())
    return idx, w, offsets, perm


def mxfp4_dequantize(blocks: torch.Tensor, scales: torch.Tensor, rows: int, cols: int,
                     status: torch.Tensor | None = None) -> torch.Tensor:
    _need(blocks, torch.uint8, "blocks")
    _need(scales, torch.uint8, "scales")
    out = torch.empty(rows, cols, dtype=torch.float32, device=blocks.device)
    call("kdq_mxfp4_dequantize", blocks.data_ptr(), scales.data_ptr(), rows, cols,
         out.data_ptr(), _ptr(status), _stream())
    return out


def moe_mxfp4(x_bf16: torch.Tensor, logits: torch.Tensor, top_k: int, gate_blocks, gate_scales,
              up_blocks, up_scales, down_blocks, down_scales, routing: bool = False,
              out: torch.Tensor | None = None):
    """The MXFP4 MoE layer (kdq_moe_mxfp4).  Returns y fp32 [tokens, hidden], plus
    (idx, w, offsets, perm) when ``routing``."""
    _need(x_bf16, torch.bfloat16, "x")
    _need(logits, torch.float32, "logits")
    t, h = x_bf16.shape
    e = logits.shape[1]
    inter = gate_scales.shape[1]
    dev = x_bf16.device
    for name, a in (("gate_blocks", gate_blocks), ("gate_scales", gate_scales),
                    ("up_blocks", up_blocks), ("up_scales", up_scales),
                    ("down_blocks", down_blocks), ("down_scales", down_scales)):
        _need(a, torch.uint8, name)
    if out is None:
        out = torch.empty(t, h, dtype=torch.float32, device=dev)
    extra = [None] * 4
    if routing:
        extra = [torch.empty(t, top_k, dtype=torch.int32, device=dev),
                 torch.empty(t, top_k, dtype=torch.float32, device=dev),
                 torch.empty(e + 1, dtype=torch.int32, device=dev),
                 torch.empty(t * top_k, dtype=torch.int32, device=dev)]
    call("kdq_moe_mxfp4", x_bf16.data_ptr(), logits.data_ptr(), t, h, inter, e, top_k,
         gate_blocks.data_ptr(), gate_scales.data_ptr(), up_blocks.data_ptr(),
         up_scales.data_ptr(), down_blocks.data_ptr(), down_scales.data_ptr(), out.data_ptr(),
         *[_ptr(a) for a in extra], _stream())
    return (out, *extra) if routing else out


def moe_mxfp4_pack(blocks: torch.Tensor, scales: torch.Tensor, experts: int, rows: int,
                   cols: int) -> torch.Tensor:
    """One projection tensor in the packed resident layout (kdq_moe_mxfp4_pack)."""
    _need(blocks, torch.uint8, "blocks")
    _need(scales, torch.uint8, "scales")
    n = lib().kdq_moe_mxfp4_packed_bytes(experts, rows, cols)
    if not n:
        raise ValueError("rows % 32 and cols % 64 must be 0")
    packed = torch.empty(n, dtype=torch.uint8, device=blocks.device)
    call("kdq_moe_mxfp4_pack", blocks.data_ptr(), scales.data_ptr(), experts, rows, cols,
         packed.data_ptr(), _stream())
    return packed


def moe_mxfp4_packed(x_bf16: torch.Tensor, logits: torch.Tensor, top_k: int, inter: int,
                     gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                     routing: bool = False, out: torch.Tensor | None = None):
    """kdq_moe_mxfp4_packed: the layer over packed weights (moe_mxfp4_pack)."""
    _need(x_bf16, torch.bfloat16, "x")
    _need(logits, torch.float32, "logits")
    t, h = x_bf16.shape
    e = logits.shape[1]
    dev = x_bf16.device
    for name, a in (("gate", gate), ("up", up), ("down", down)):
        _need(a, torch.uint8, name)
    if out is None:
        out = torch.empty(t, h, dtype=torch.float32, device=dev)
    extra = [None] * 4
    if routing:
        extra = [torch.empty(t, top_k, dtype=torch.int32, device=dev),
                 torch.empty(t, top_k, dtype=torch.float32, device=dev),
                 torch.empty(e + 1, dtype=torch.int32, device=dev),
                 torch.empty(t * top_k, dtype=torch.int32, device=dev)]
    call("kdq_moe_mxfp4_packed", x_bf16.data_ptr(), logits.data_ptr(), t, h, inter, e, top_k,
         gate.data_ptr(), up.data_ptr(), down.data_ptr(), out.data_ptr(),
         *[_ptr(a) for a in extra], _stream())
    return (out, *extra) if routing else out


def _stream_for(*tensors: torch.Tensor) -> int:
    """The current device's current stream, where every tensor is on that device."""
    device = _current_device()
    for t in tensors:
        if t.get_device() != device:
            raise ValueError("every tensor must be on the current device")
    return (torch.cuda.current_stream().cuda_stream if _raw_stream is None
            else _raw_stream(device))


def _row_stride(t: torch.Tensor, dtype, name: str, multiple: int = 8) -> int:
    """Values from row to row of a 2-d device tensor whose rows are contiguous."""
    if t.dtype != dtype or t.dim() != 2 or not t.is_cuda:
        raise ValueError(f"{name}: expected a 2-d {dtype} device tensor")
    rows, cols = t.shape
    row, col = t.stride()
    if cols > 1 and col != 1:
        raise ValueError(f"{name}: values of a row must lie side by side")
    if rows == 1:
        return cols
    if row < cols or row % multiple:
        raise ValueError(f"{name}: rows must not overlap and lie a multiple of {multiple} "
                         "values apart")
    return row


def _no_graph(t: torch.Tensor, name: str) -> None:
    """Refuses a tensor whose gradient would be lost: the calls record none."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this call does not record: make it "
                         "under torch.no_grad(), or within a torch.autograd.Function")


_BF16 = torch.bfloat16
_TYPES = {torch.float32: 0, torch.float16: 1, _BF16: 30}  # KDQ_F32, KDQ_F16, KDQ_BF16


def _type(dtype) -> int:
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"no MXFP4 operator takes {dtype}")
    return kind


def _blocks(blocks: torch.Tensor, scales: torch.Tensor) -> tuple[int, int]:
    """Rows and values of a row of an MXFP4 matrix."""
    _need(blocks, torch.uint8, "blocks")
    _need(scales, torch.uint8, "scales")
    if blocks.dim() == 2 and scales.dim() == 2:
        rows, width = blocks.shape
        if scales.shape == (rows, width // 16) and width % 16 == 0:
            return rows, 2 * width
    raise ValueError("expected blocks [rows, cols/2] and scales [rows, cols/32]")


# Device bytes that a call's matrices and workspace take.  (A decode product takes 6-8 us on
# the device and its wrapper must not take longer, so they are asked for once.)
@functools.lru_cache(maxsize=4096, typed=True)
def _mxfp4_size(function: str, *sizes: int) -> int:
    return int(getattr(lib(), function)(*sizes))


@functools.lru_cache(maxsize=4096, typed=True)
def _mxfp4_sizes_on(device: int, matrix: str, rows: int, cols: int, workspace: str, *sizes: int):
    return _mxfp4_size(matrix, rows, cols), int(getattr(lib(), workspace)(*sizes))


def _mxfp4_sizes(*sizes):
    """The matrix's bytes and the workspace's, which depend on the current device's compute
    units."""
    return _mxfp4_sizes_on(_current_device(), *sizes)


@functools.lru_cache(maxsize=4096, typed=True)
def _experts_sizes_on(device: int, stack: str, experts: int, rows: int, cols: int, workspace: str,
                      *sizes: int):
    return _mxfp4_size(stack, experts, rows, cols), int(getattr(lib(), workspace)(*sizes))


def _experts_sizes(*sizes):
    """The same for a stack of experts' matrices."""
    return _experts_sizes_on(_current_device(), *sizes)


_PACKED, _TRANSPOSED = "kdq_mxfp4_packed_bytes", "kdq_mxfp4_packed_transposed_bytes"
_EXPERTS = "kdq_mxfp4_experts_packed_bytes"
_EXPERTS_TRANSPOSED = "kdq_mxfp4_experts_packed_transposed_bytes"


# The two packed forms of a matrix may take the same number of bytes (14336 x 4096 does), so
# they are told apart by their shape: flat for the products, a row per 64 columns transposed.
def _matrix(packed: torch.Tensor, size: int, name: str, dims: int = 1) -> int:
    if packed.dtype != torch.uint8 or not packed.is_cuda or not packed.is_contiguous():
        raise ValueError(f"{name}: expected a packed uint8 device tensor")
    if not size or packed.numel() != size:
        raise ValueError(f"{name}: not the packed size of this call's matrix")
    if packed.dim() != dims:
        raise ValueError(f"{name}: expected mxfp4_pack's flat form" if dims == 1 else
                         f"{name}: expected the form of mxfp4_pack(..., transposed=True)" +
                         (" of a stack" if dims == 3 else ""))
    return packed.data_ptr()


def _transposed_matrix(packed: torch.Tensor, size: int, cols: int, name: str) -> int:
    at = _matrix(packed, size, name, 2)
    if packed.shape[0] != (cols + 63) // 64:
        raise ValueError(f"{name}: another matrix's packed form")
    return at


def _output(out: torch.Tensor, rows: int, cols: int, dtype, name: str) -> int:
    """Values from row to row of a given output."""
    if out.dim() != 2 or out.shape[0] != rows or out.shape[1] != cols:
        raise ValueError(f"{name}: expected [{rows}, {cols}]")
    return _row_stride(out, dtype, name, 1)


def _scratch(size: int, device) -> torch.Tensor | None:
    """A call's workspace: torch's allocator keeps it to the current stream (and to a
    graph's own pool under capture), so calls share none.  Keep it until the call is
    enqueued."""
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def mxfp4_quantize(x: torch.Tensor, status: torch.Tensor | None = None):
    """fp32, fp16 or bf16 [rows, cols] (cols % 32 == 0) as MXFP4: blocks uint8
    [rows, cols/2] and scales uint8 [rows, cols/32]; ``status``, an int32, is set to 1 where
    a value is not finite (kdq_mxfp4_quantize)."""
    if status is None:
        flag, parts = None, (x,)
    else:
        _need(status, torch.int32, "status")
        if not status.numel():
            raise ValueError("status: expected one value")
        flag, parts = status.data_ptr(), (x, status)
    dtype = x.dtype
    kind = _type(dtype)
    stride = _row_stride(x, dtype, "x")
    stream = _stream_for(*parts)
    rows, cols = x.shape
    if cols % 32:
        raise ValueError("x: a row must be whole blocks of 32 values")
    device = x.device
    blocks = torch.empty(rows, cols // 2, dtype=torch.uint8, device=device)
    scales = torch.empty(rows, cols // 32, dtype=torch.uint8, device=device)
    call("kdq_mxfp4_quantize", kind, x.data_ptr(), stride, rows, cols, blocks.data_ptr(),
         scales.data_ptr(), flag, stream)
    return blocks, scales


def mxfp4_pack(blocks: torch.Tensor, scales: torch.Tensor,
               transposed: bool = False) -> torch.Tensor:
    """An MXFP4 matrix in the form the products read, uint8 [bytes] (kdq_mxfp4_pack), or,
    ``transposed``, in the one that the backward passes read, uint8 [ceil(cols / 64), bytes of
    64 columns] (kdq_mxfp4_pack_transposed).  The shape is what tells the two forms apart; of
    matrices of other sizes the calls see the number of bytes alone.  A stack of experts' matrices
    (blocks and scales with a first dimension of experts) gives the experts' forms: uint8 [bytes],
    which for rows of whole 32s and cols of whole 64s is moe_mxfp4_pack's, and uint8 [experts,
    ceil(cols / 64), bytes] (kdq_mxfp4_experts_pack, kdq_mxfp4_experts_pack_transposed)."""
    if blocks.dim() == 3:
        return _pack_experts(blocks, scales, transposed)
    rows, cols = _blocks(blocks, scales)
    stream = _stream_for(blocks, scales)
    size = _mxfp4_size(_TRANSPOSED if transposed else _PACKED, rows, cols)
    if not size:
        raise ValueError(f"a matrix of {rows} x {cols} has no packed form")
    groups = (cols + 63) // 64
    packed = torch.empty((groups, size // groups) if transposed else size, dtype=torch.uint8,
                         device=blocks.device)
    call("kdq_mxfp4_pack_transposed" if transposed else "kdq_mxfp4_pack", blocks.data_ptr(),
         scales.data_ptr(), rows, cols, packed.data_ptr(), stream)
    return packed


def _pack_experts(blocks: torch.Tensor, scales: torch.Tensor, transposed: bool) -> torch.Tensor:
    _need(blocks, torch.uint8, "blocks")
    _need(scales, torch.uint8, "scales")
    experts, rows, width = blocks.shape
    if scales.shape != (experts, rows, width // 16) or width % 16:
        raise ValueError("expected blocks [experts, rows, cols/2], scales [experts, rows, cols/32]")
    cols = 2 * width
    stream = _stream_for(blocks, scales)
    size = _mxfp4_size(_EXPERTS_TRANSPOSED if transposed else _EXPERTS, experts, rows, cols)
    if not size:
        raise ValueError(f"{experts} matrices of {rows} x {cols} have no packed form")
    groups = (cols + 63) // 64
    packed = torch.empty((experts, groups, size // (experts * groups)) if transposed else size,
                         dtype=torch.uint8, device=blocks.device)
    call("kdq_mxfp4_experts_pack_transposed" if transposed else "kdq_mxfp4_experts_pack",
         blocks.data_ptr(), scales.data_ptr(), experts, rows, cols, packed.data_ptr(), stream)
    return packed


def mxfp4_product(x: torch.Tensor, packed: torch.Tensor, n_out: int,
                  dtype: torch.dtype = torch.float32,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [m, k] times a packed MXFP4 matrix (mxfp4_pack) of n_out rows of k values ->
    fp32 or bf16 [m, n_out] (kdq_mxfp4_product)."""
    _no_graph(x, "x")
    stride = _row_stride(x, _BF16, "x")
    m, k = x.shape
    kind = _type(dtype)
    weights, size = _mxfp4_sizes(_PACKED, n_out, k, "kdq_mxfp4_product_workspace", m, n_out, k, 0)
    w = _matrix(packed, weights, "packed")
    if out is None:
        stream, y_stride = _stream_for(x, packed), n_out
        out = torch.empty(m, n_out, dtype=dtype, device=x.device)
    else:
        y_stride = _output(out, m, n_out, dtype, "out")
        stream = _stream_for(x, packed, out)
    scratch = _scratch(size, x.device)
    call("kdq_mxfp4_product", x.data_ptr(), stride, m, w, n_out, k, kind, out.data_ptr(),
         y_stride, _ptr(scratch), size, stream)
    return out


def mxfp4_product_quantized(blocks: torch.Tensor, scales: torch.Tensor, packed: torch.Tensor,
                            n_out: int, dtype: torch.dtype = torch.float32,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """MXFP4 activations (mxfp4_quantize) times a packed MXFP4 matrix of n_out rows -> fp32
    or bf16 [m, n_out] (kdq_mxfp4_product_quantized)."""
    m, k = _blocks(blocks, scales)
    kind = _type(dtype)
    weights, size = _mxfp4_sizes(_PACKED, n_out, k, "kdq_mxfp4_product_workspace", m, n_out, k, 1)
    w = _matrix(packed, weights, "packed")
    if out is None:
        stream, y_stride = _stream_for(blocks, scales, packed), n_out
        out = torch.empty(m, n_out, dtype=dtype, device=blocks.device)
    else:
        y_stride = _output(out, m, n_out, dtype, "out")
        stream = _stream_for(blocks, scales, packed, out)
    scratch = _scratch(size, blocks.device)
    call("kdq_mxfp4_product_quantized", blocks.data_ptr(), scales.data_ptr(), m, w, n_out, k,
         kind, out.data_ptr(), y_stride, _ptr(scratch), size, stream)
    return out


def mxfp4_gated(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, n_out: int,
                save: str | None = None, out: torch.Tensor | None = None):
    """h = silu(x Wg^T) * (x Wu^T): bf16 [m, k] and two packed MXFP4 matrices (mxfp4_pack) of
    n_out rows (n_out % 32 == 0) -> bf16 [m, n_out] (kdq_mxfp4_gated).  With ``save`` the
    pre-activations are kept for mxfp4_gated_backward, and (h, saved) returned: "bf16" as one
    tensor [m, 2 n_out], "q8" as int8 [m, 2 n_out] and fp32 scales [m, 2 n_out / 32].  Nothing
    is recorded for autograd: the two calls are the halves of a torch.autograd.Function."""
    _no_graph(x, "x")
    stride = _row_stride(x, _BF16, "x")
    if save not in (None, "bf16", "q8"):
        raise ValueError('save: None, "bf16" or "q8"')
    m, k = x.shape
    if n_out % 32:
        raise ValueError("n_out must be a multiple of 32")
    weights, size = _mxfp4_sizes(_PACKED, n_out, k, "kdq_mxfp4_gated_workspace", m, n_out, k,
                                 0 if save is None else 1)
    wg, wu = _matrix(gate, weights, "gate"), _matrix(up, weights, "up")
    device = x.device
    if out is None:
        stream, h_stride = _stream_for(x, gate, up), n_out
        out = torch.empty(m, n_out, dtype=_BF16, device=device)
    else:
        h_stride = _output(out, m, n_out, _BF16, "out")
        stream = _stream_for(x, gate, up, out)
    saved = kept = codes = scales = None
    if save == "bf16":
        saved = torch.empty(m, 2 * n_out, dtype=_BF16, device=device)
        kept = saved.data_ptr()
    elif save == "q8":
        saved = (torch.empty(m, 2 * n_out, dtype=torch.int8, device=device),
                 torch.empty(m, n_out // 16, dtype=torch.float32, device=device))
        codes, scales = saved[0].data_ptr(), saved[1].data_ptr()
    scratch = _scratch(size, device)
    call("kdq_mxfp4_gated", x.data_ptr(), stride, m, wg, wu, n_out, k, out.data_ptr(), h_stride,
         kept, codes, scales, _ptr(scratch), size, stream)
    return out if save is None else (out, saved)


def mxfp4_gated_backward(dh: torch.Tensor, saved, gate: torch.Tensor, up: torch.Tensor,
                         n_in: int, out: torch.Tensor | None = None):
    """The backward pass of mxfp4_gated over frozen weights: dh bf16 [m, n_out], ``saved``
    from its forward pass, the matrices from mxfp4_pack(..., transposed=True) -> dx bf16
    [m, n_in] and the pre-activations' gradients bf16 [m, 2 n_out], gates then ups
    (kdq_mxfp4_gated_backward)."""
    _no_graph(dh, "dh")
    stride = _row_stride(dh, _BF16, "dh")
    m, n = dh.shape
    if n % 32 or n_in % 32 or not n_in:
        raise ValueError("n_out and n_in must be multiples of 32")
    weights, size = _mxfp4_sizes(_TRANSPOSED, n, n_in, "kdq_mxfp4_gated_backward_workspace", m,
                                 n, n_in)
    wg = _transposed_matrix(gate, weights, n_in, "gate")
    wu = _transposed_matrix(up, weights, n_in, "up")
    parts, (kept, codes, scales) = _saved_gates(saved, m, n)
    device = dh.device
    if out is None:
        stream, dx_stride = _stream_for(dh, gate, up, *parts), n_in
        out = torch.empty(m, n_in, dtype=_BF16, device=device)
    else:
        dx_stride = _output(out, m, n_in, _BF16, "out")
        stream = _stream_for(dh, gate, up, out, *parts)
    dgu = torch.empty(m, 2 * n, dtype=_BF16, device=device)
    scratch = _scratch(size, device)
    call("kdq_mxfp4_gated_backward", dh.data_ptr(), stride, m, kept, codes, scales, wg, wu, n,
         n_in, dgu.data_ptr(), out.data_ptr(), dx_stride, _ptr(scratch), size, stream)
    return out, dgu


_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}  # KDQ_ACT_NONE, _SILU, _GELU
_GATES = {"silu": 1, "clamped": 3}              # KDQ_ACT_SILU, _CLAMPED


def _activation(kinds: dict, activation) -> int:
    if activation not in kinds:
        raise ValueError(f"activation: one of {', '.join(map(repr, kinds))}")
    return kinds[activation]


def _offsets(offsets: torch.Tensor) -> int:
    """The number of experts."""
    _need(offsets, torch.int32, "offsets")
    experts = offsets.numel() - 1
    if offsets.dim() != 1 or not 1 <= experts <= 256:
        raise ValueError("offsets: expected 1 to 256 experts' offsets and the end of the last")
    return experts


def _bias(bias: torch.Tensor, name: str, shape: tuple) -> int:
    _no_graph(bias, name)
    if (bias.dtype != torch.float32 or bias.shape != shape or not bias.is_contiguous()
            or bias.get_device() != _current_device()):
        raise ValueError(f"{name}: expected a contiguous fp32 tensor of {list(shape)} on the "
                         "current device")
    return bias.data_ptr()


def _here(t: torch.Tensor, name: str) -> None:
    if t.get_device() != _current_device():
        raise ValueError(f"{name}: expected on the current device")


def _transposed_stack(packed: torch.Tensor, size: int, experts: int, cols: int, name: str) -> int:
    at = _matrix(packed, size, name, 3)
    if packed.shape[:2] != (experts, (cols + 63) // 64):
        raise ValueError(f"{name}: another stack's packed form")
    return at


def mxfp4_linear(x: torch.Tensor, packed: torch.Tensor, n_out: int,
                 bias: torch.Tensor | None = None, activation: str | None = None,
                 residual: torch.Tensor | None = None, dtype: torch.dtype = torch.float32,
                 offsets: torch.Tensor | None = None, save: bool = False,
                 out: torch.Tensor | None = None):
    """y = residual + act(x W^T + bias): bf16 [m, k] and a packed MXFP4 matrix (mxfp4_pack) of
    n_out rows -> fp32 or bf16 [m, n_out], with a bias fp32 [n_out], an activation (None, "silu"
    or "gelu", the tanh form) and a residual of y's type, each or none of them (``out`` may be the
    residual itself).  With ``offsets`` int32 [experts + 1] (moe_route's) the rows are sorted by
    expert (moe_sort) and each is multiplied by its own expert's matrix of a packed stack, with
    its bias of [experts, n_out]; rows that no expert has are left as they are in ``out`` (and are
    undefined in a new tensor, and in what is saved).  With ``save`` the pre-activations are kept
    for mxfp4_linear_backward, bf16 [m, n_out], and (y, saved) returned.  Nothing is recorded for
    autograd (kdq_mxfp4_linear)."""
    _no_graph(x, "x")
    stride = _row_stride(x, _BF16, "x")
    kind, act = _type(dtype), _activation(_ACTIVATIONS, activation)
    if save and not act:
        raise ValueError("save: without an activation there is nothing to keep")
    m, k = x.shape
    if offsets is None:
        experts, table = 1, None
        weights, size = _mxfp4_sizes(_PACKED, n_out, k, "kdq_mxfp4_linear_workspace", m, 0, n_out,
                                     k)
        w = _matrix(packed, weights, "packed")
        stream = _stream_for(x, packed)
    else:
        experts, table = _offsets(offsets), offsets.data_ptr()
        weights, size = _experts_sizes(_EXPERTS, experts, n_out, k, "kdq_mxfp4_linear_workspace", m,
                                       experts, n_out, k)
        w = _matrix(packed, weights, "packed")
        stream = _stream_for(x, packed, offsets)
    b = add = None
    if bias is not None:
        b = _bias(bias, "bias", (n_out,) if table is None else (experts, n_out))
    add_stride = 0
    if residual is not None:
        _no_graph(residual, "residual")
        add, add_stride = residual.data_ptr(), _output(residual, m, n_out, dtype, "residual")
        _here(residual, "residual")
    if out is None:
        y_stride, out = n_out, x.new_empty(m, n_out, dtype=dtype)
    else:
        y_stride = _output(out, m, n_out, dtype, "out")
        _here(out, "out")
    saved = x.new_empty(m, n_out) if save else None
    scratch = _scratch(size, x.device) if size else None
    call("kdq_mxfp4_linear", x.data_ptr(), stride, m, table, experts, w, n_out, k, b, act, add,
         add_stride, kind, out.data_ptr(), y_stride, _ptr(saved), _ptr(scratch), size, stream)
    return (out, saved) if save else out


def mxfp4_linear_backward(dy: torch.Tensor, packed: torch.Tensor, n_in: int,
                          saved: torch.Tensor | None = None, activation: str | None = None,
                          offsets: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """The backward pass of mxfp4_linear over frozen weights: dy bf16 [m, n_out]
    (n_out % 8 == 0), with an activation what its forward pass saved, and the matrix or stack from
    mxfp4_pack(..., transposed=True) -> dx bf16 [m, n_in] and dpre bf16 [m, n_out], the gradient
    before the activation (dy itself without one; the bias's gradient is the sum of its rows, an
    expert's of its own rows).  Of rows that no expert has dx is left as it is in ``out`` (undefined
    in a new tensor) and dpre undefined (kdq_mxfp4_linear_backward)."""
    _no_graph(dy, "dy")
    stride = _row_stride(dy, _BF16, "dy")
    act = _activation(_ACTIVATIONS, activation)
    m, n = dy.shape
    if n % 8 or n_in % 32 or not n_in:
        raise ValueError("n_out must be a multiple of 8, n_in of 32")
    if (saved is None) == bool(act):
        raise ValueError("saved: expected with an activation, and only with one")
    parts = [dy, packed]
    if offsets is None:
        experts, table = 1, None
        weights, size = _mxfp4_sizes(_TRANSPOSED, n, n_in, "kdq_mxfp4_linear_backward_workspace",
                                     m, 0, n, n_in)
        w = _transposed_matrix(packed, weights, n_in, "packed")
    else:
        experts, table = _offsets(offsets), offsets.data_ptr()
        weights, size = _experts_sizes(_EXPERTS_TRANSPOSED, experts, n, n_in,
                                       "kdq_mxfp4_linear_backward_workspace", m, experts, n, n_in)
        w = _transposed_stack(packed, weights, experts, n_in, "packed")
        parts.append(offsets)
    device = dy.device
    dpre = dy
    if act:
        _need(saved, _BF16, "saved")
        if saved.shape != (m, n):
            raise ValueError("saved: of another shape than dy")
        parts.append(saved)
        dpre = torch.empty(m, n, dtype=_BF16, device=device)
    if out is None:
        stream, dx_stride = _stream_for(*parts), n_in
        out = torch.empty(m, n_in, dtype=_BF16, device=device)
    else:
        dx_stride = _output(out, m, n_in, _BF16, "out")
        stream = _stream_for(*parts, out)
    scratch = _scratch(size, device)
    call("kdq_mxfp4_linear_backward", dy.data_ptr(), stride, m, table, experts, _ptr(saved), act,
         w, n, n_in, dpre.data_ptr() if act else None, out.data_ptr(), dx_stride, _ptr(scratch),
         size, stream)
    return out, dpre


def mxfp4_experts_gated(x: torch.Tensor, offsets: torch.Tensor, gate: torch.Tensor,
                        up: torch.Tensor, n_out: int, gate_bias: torch.Tensor | None = None,
                        up_bias: torch.Tensor | None = None, activation: str = "silu",
                        save: str | None = None, out: torch.Tensor | None = None):
    """mxfp4_gated of a mixture's experts: bf16 [m, k] rows sorted by expert (moe_sort), offsets
    int32 [experts + 1] (moe_route's) and two packed stacks (mxfp4_pack) of n_out rows
    (n_out % 32 == 0), with biases fp32 [experts, n_out] or none -> h bf16 [m, n_out]:
    silu(g) * u, or, "clamped", with g' = min(g, 7) and u' = u between -7 and 7,
    g' sigmoid(1.702 g') (u' + 1).  Rows that no expert has are left as they are in ``out`` (and are
    undefined in a new tensor, and in what is saved).  ``save`` as for mxfp4_gated.  Nothing is
    recorded for autograd (kdq_mxfp4_experts_gated)."""
    _no_graph(x, "x")
    stride = _row_stride(x, _BF16, "x")
    act = _activation(_GATES, activation)
    if save not in (None, "bf16", "q8"):
        raise ValueError('save: None, "bf16" or "q8"')
    if n_out % 32:
        raise ValueError("n_out must be a multiple of 32")
    if (gate_bias is None) != (up_bias is None):
        raise ValueError("expected both biases or none")
    m, k = x.shape
    experts = _offsets(offsets)
    weights, size = _experts_sizes(_EXPERTS, experts, n_out, k, "kdq_mxfp4_experts_gated_workspace",
                                   m, experts, n_out, k, 0 if save is None else 1)
    wg, wu = _matrix(gate, weights, "gate"), _matrix(up, weights, "up")
    stream = _stream_for(x, offsets, gate, up)
    bg = bu = None
    if gate_bias is not None:
        bg = _bias(gate_bias, "gate_bias", (experts, n_out))
        bu = _bias(up_bias, "up_bias", (experts, n_out))
    if out is None:
        h_stride, out = n_out, x.new_empty(m, n_out)
    else:
        h_stride = _output(out, m, n_out, _BF16, "out")
        _here(out, "out")
    saved = kept = codes = scales = None
    if save == "bf16":
        saved = x.new_empty(m, 2 * n_out)
        kept = saved.data_ptr()
    elif save == "q8":
        saved = (x.new_empty(m, 2 * n_out, dtype=torch.int8),
                 x.new_empty(m, n_out // 16, dtype=torch.float32))
        codes, scales = saved[0].data_ptr(), saved[1].data_ptr()
    scratch = _scratch(size, x.device) if size else None
    call("kdq_mxfp4_experts_gated", x.data_ptr(), stride, m, offsets.data_ptr(), experts, wg, wu,
         n_out, k, bg, bu, act, out.data_ptr(), h_stride, kept, codes, scales, _ptr(scratch), size,
         stream)
    return out if save is None else (out, saved)


def _saved_gates(saved, m: int, n: int):
    """Kept pre-activations: the tensors, and the pointers to bf16 values, codes and scales."""
    if isinstance(saved, torch.Tensor):
        _need(saved, _BF16, "saved")
        parts, at = (saved,), (saved.data_ptr(), None, None)
    else:
        parts = q, d = saved
        _need(q, torch.int8, "saved codes")
        _need(d, torch.float32, "saved scales")
        if d.shape != (m, n // 16):
            raise ValueError("saved: scales of another shape")
        at = (None, q.data_ptr(), d.data_ptr())
    if parts[0].shape != (m, 2 * n):
        raise ValueError("saved: of another shape than dh")
    return parts, at


def mxfp4_experts_gated_backward(dh: torch.Tensor, offsets: torch.Tensor, saved,
                                 gate: torch.Tensor, up: torch.Tensor, n_in: int,
                                 activation: str = "silu", out: torch.Tensor | None = None):
    """The backward pass of mxfp4_experts_gated over frozen weights: dh bf16 [m, n_out], its
    offsets, ``saved`` from its forward pass, the stacks from mxfp4_pack(..., transposed=True)
    -> dx bf16 [m, n_in] and the pre-activations' gradients bf16 [m, 2 n_out], gates then ups.  Of
    rows that no expert has dx is left as it is in ``out`` (undefined in a new tensor) and the
    gradients undefined (kdq_mxfp4_experts_gated_backward)."""
    _no_graph(dh, "dh")
    stride = _row_stride(dh, _BF16, "dh")
    act = _activation(_GATES, activation)
    m, n = dh.shape
    if n % 32 or n_in % 32 or not n_in:
        raise ValueError("n_out and n_in must be multiples of 32")
    experts = _offsets(offsets)
    weights, size = _experts_sizes(_EXPERTS_TRANSPOSED, experts, n, n_in,
                                   "kdq_mxfp4_experts_gated_backward_workspace", m, experts, n,
                                   n_in)
    wg = _transposed_stack(gate, weights, experts, n_in, "gate")
    wu = _transposed_stack(up, weights, experts, n_in, "up")
    parts, (kept, codes, scales) = _saved_gates(saved, m, n)
    device = dh.device
    if out is None:
        stream, dx_stride = _stream_for(dh, offsets, gate, up, *parts), n_in
        out = torch.empty(m, n_in, dtype=_BF16, device=device)
    else:
        dx_stride = _output(out, m, n_in, _BF16, "out")
        stream = _stream_for(dh, offsets, gate, up, out, *parts)
    dgu = torch.empty(m, 2 * n, dtype=_BF16, device=device)
    scratch = _scratch(size, device)
    call("kdq_mxfp4_experts_gated_backward", dh.data_ptr(), stride, m, offsets.data_ptr(),
         experts, kept, codes, scales, act, wg, wu, n, n_in, dgu.data_ptr(), out.data_ptr(),
         dx_stride, _ptr(scratch), size, stream)
    return out, dgu


# (A few tokens' rows take 2-4 us on the device, their wrappers more than that: so few steps.)
_F32, _I32 = torch.float32, torch.int32


def _rows_of(t: torch.Tensor, name: str) -> tuple[int, int]:
    """KDQ type of fp32, fp16 or bf16 rows, and the values from row to row."""
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name}: expected fp32, fp16 or bf16 rows")
    if t.is_contiguous() and t.dim() == 2:
        return kind, t.shape[1]
    return kind, _row_stride(t, t.dtype, name, 1)


def _slots(t: torch.Tensor, slots: int, name: str) -> int:
    """A contiguous int32 tensor of a value per slot."""
    if t.dtype != _I32 or not t.is_cuda or not t.is_contiguous() or t.numel() != slots:
        raise ValueError(f"{name}: expected a contiguous int32 device tensor of {slots} values, "
                         "one per selection")
    return t.data_ptr()


def moe_sort(x: torch.Tensor, perm: torch.Tensor, top_k: int):
    """Tokens sorted by expert: x [tokens, cols] (fp32, fp16 or bf16) and moe_route's perm ->
    rows [tokens * top_k, cols], rows[p] = x[perm[p] // top_k], and place int32
    [tokens * top_k], place[perm[p]] = p.  An entry of perm that is no slot (-1, say) gives a row of
    zeros, and a slot that perm does not name the place -1: a dropped selection, which the calls
    that take place leave out (kdq_moe_sort).  Nothing is recorded for autograd: its backward pass
    is moe_sort_backward."""
    if x.requires_grad:
        _no_graph(x, "x")
    kind, stride = _rows_of(x, "x")
    tokens, cols = x.shape
    slots = tokens * top_k
    order = _slots(perm, slots, "perm")
    stream = _stream_for(x, perm)
    rows, place = x.new_empty(slots, cols), torch.empty_like(perm)
    call("kdq_moe_sort", kind, x.data_ptr(), stride, tokens, cols, top_k, order, rows.data_ptr(),
         cols, place.data_ptr(), stream)
    return rows, place


def moe_sort_backward(drows: torch.Tensor, place: torch.Tensor, top_k: int) -> torch.Tensor:
    """The gradient of moe_sort: drows [tokens * top_k, cols] -> dx [tokens, cols] of its type,
    each token's rows summed (kdq_moe_sort_backward)."""
    if drows.requires_grad:
        _no_graph(drows, "drows")
    kind, stride = _rows_of(drows, "drows")
    slots, cols = drows.shape
    if top_k < 1 or slots % top_k:
        raise ValueError("drows: expected top_k rows per token")
    at = _slots(place, slots, "place")
    stream = _stream_for(drows, place)
    dx = drows.new_empty(slots // top_k, cols)
    call("kdq_moe_sort_backward", kind, drows.data_ptr(), stride, at, slots // top_k, cols, top_k,
         dx.data_ptr(), cols, stream)
    return dx


def _weights(weights: torch.Tensor) -> tuple[int, int]:
    if (weights.dtype != _F32 or not weights.is_cuda or weights.dim() != 2
            or not weights.is_contiguous()):
        raise ValueError("weights: expected a contiguous fp32 device tensor [tokens, top_k]")
    return weights.shape


def moe_combine(rows: torch.Tensor, weights: torch.Tensor, place: torch.Tensor,
                residual: torch.Tensor | None = None, dtype: torch.dtype | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """Experts' rows back to their tokens: y[t] = residual[t] + sum_i weights[t, i] *
    rows[place[t * top_k + i]], rows [tokens * top_k, cols] (fp32, fp16 or bf16), weights fp32
    [tokens, top_k], place from moe_sort -> y [tokens, cols] of the rows' type or fp32
    (``dtype``; the residual's, and ``out`` may be the residual itself) (kdq_moe_combine).
    Nothing is recorded for autograd: its backward pass is moe_combine_backward."""
    if rows.requires_grad:
        _no_graph(rows, "rows")
    if weights.requires_grad:
        _no_graph(weights, "weights")
    kind, stride = _rows_of(rows, "rows")
    tokens, top_k = _weights(weights)
    slots, cols = rows.shape
    if slots != tokens * top_k:
        raise ValueError("rows: expected one per weight")
    at = _slots(place, slots, "place")
    if dtype is None:
        dtype = rows.dtype
    if dtype != rows.dtype and dtype != torch.float32:
        raise ValueError("dtype: the rows' type or fp32")
    stream = _stream_for(rows, weights, place)
    add, add_stride = None, 0
    if residual is not None:
        if residual.requires_grad:
            _no_graph(residual, "residual")
        add, add_stride = residual.data_ptr(), _output(residual, tokens, cols, dtype, "residual")
        _here(residual, "residual")
    if out is None:
        y_stride, out = cols, rows.new_empty(tokens, cols, dtype=dtype)
    else:
        y_stride = _output(out, tokens, cols, dtype, "out")
        _here(out, "out")
    call("kdq_moe_combine", kind, rows.data_ptr(), stride, at, weights.data_ptr(), tokens, cols,
         top_k, _TYPES[dtype], add, add_stride, out.data_ptr(), y_stride, stream)
    return out


def moe_combine_backward(dy: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor,
                         place: torch.Tensor):
    """The gradients of moe_combine: dy [tokens, cols] (the rows' type or fp32) and its rows,
    weights and place -> drows [tokens * top_k, cols] of the rows' type and dweights fp32
    [tokens, top_k] (kdq_moe_combine_backward); zeros for dropped selections (places of -1) and for
    the rows that no place names.  The residual's gradient is dy."""
    if dy.requires_grad:
        _no_graph(dy, "dy")
    kind, stride = _rows_of(rows, "rows")
    dy_kind, dy_stride = _rows_of(dy, "dy")
    if dy_kind not in (kind, 0):
        raise ValueError("dy: the rows' type or fp32")
    tokens, top_k = _weights(weights)
    slots, cols = rows.shape
    if slots != tokens * top_k or dy.shape != (tokens, cols):
        raise ValueError("expected rows [tokens * top_k, cols] and dy [tokens, cols]")
    at = _slots(place, slots, "place")
    stream = _stream_for(rows, weights, place, dy)
    drows, dweights = rows.new_empty(slots, cols), weights.new_empty(tokens, top_k)
    call("kdq_moe_combine_backward", kind, rows.data_ptr(), stride, at, weights.data_ptr(),
         tokens, cols, top_k, dy_kind, dy.data_ptr(), dy_stride, drows.data_ptr(), cols,
         dweights.data_ptr(), stream)
    return drows, dweights


def moe_route_backward(idx: torch.Tensor, weights: torch.Tensor, dweights: torch.Tensor,
                       experts: int) -> torch.Tensor:
    """The gradient of moe_route's weights: idx int32, weights and their gradient fp32, each
    [tokens, top_k] -> dlogits fp32 [tokens, experts] (kdq_moe_route_backward)."""
    if dweights.requires_grad:
        _no_graph(dweights, "dweights")
    tokens, top_k = _weights(weights)
    if (idx.dtype != _I32 or dweights.dtype != _F32 or idx.shape != weights.shape
            or dweights.shape != weights.shape or not idx.is_contiguous()
            or not dweights.is_contiguous()):
        raise ValueError("expected contiguous idx int32 and dweights fp32 of the weights' shape")
    stream = _stream_for(idx, weights, dweights)
    dlogits = weights.new_empty(tokens, experts)
    call("kdq_moe_route_backward", idx.data_ptr(), weights.data_ptr(), dweights.data_ptr(), tokens,
         experts, top_k, dlogits.data_ptr(), stream)
    return dlogits


def hbm_read(buffer: torch.Tensor, sink: torch.Tensor, workgroups: int,
             threads: int = 256, store_all: bool = True, match: int = 0) -> None:
    """kdq_hbm_read: one streaming read of `buffer` (the HBM read ceiling's probe) over
    `workgroups` workgroups of `threads` lanes; `sink` holds one int32 per workgroup,
    written always (store_all) or where the workgroup's fold equals `match`."""
    _need(sink, torch.int32, "sink")
    if not buffer.is_cuda or not buffer.is_contiguous() or sink.numel() < workgroups:
        raise ValueError("hbm_read: a contiguous device buffer and a sink per workgroup")
    call("kdq_hbm_read", buffer.data_ptr(), buffer.numel() * buffer.element_size(),
         sink.data_ptr(), workgroups, threads, int(store_all), match & 0xFFFFFFFF, _stream())


__all__ = ["dequantize", "gemv", "gemv_batch", "quantize_q8", "gemm_q4_0", "gemm_q4_0_packed",
           "gemm_packed", "hbm_read",
           "moe_gguf", "moe_route",
           "mxfp4_quantize", "mxfp4_pack", "mxfp4_product", "mxfp4_product_quantized",
           "mxfp4_gated", "mxfp4_gated_backward",
           "moe_sort", "moe_sort_backward", "moe_combine", "moe_combine_backward",
           "moe_route_backward", "mxfp4_linear", "mxfp4_linear_backward", "mxfp4_experts_gated",
           "mxfp4_experts_gated_backward",
           "mxfp4_dequantize", "moe_mxfp4", "moe_mxfp4_pack", "moe_mxfp4_packed", "lib",
           "BLOCK_BYTES", "BLOCK_VALUES"]
