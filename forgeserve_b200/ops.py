"""Tensor-level wrappers of the C ABI: each function checks its torch tensors (CUDA, dtype, layout), passes raw
pointers and the caller's current CUDA stream to libforgeserve_b200.so, and returns torch tensors it allocated
(the caller owns them). Nothing here computes on the CPU."""

import ctypes
import math
import struct
from typing import List, Optional

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.FS_F32, torch.bfloat16: L.FS_BF16}

# When set to a list, every projection GEMM appends (start_event, end_event, flops) recorded on its stream.
gemm_events: Optional[List] = None


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise TypeError(f"forgeserve_b200 kernels support float32 and bfloat16, not {dtype}") from None


def require_cuda(*tensors) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "forgeserve_b200 runs its path as CUDA kernels only (no CPU fallback); "
                f"got a tensor on {t.device}. Move the module and inputs to a CUDA device.")


def _p(t: Optional[torch.Tensor]) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _rows(t: torch.Tensor):
    """View a (..., n) tensor whose last dim is contiguous as rows: returns (num_rows, row_stride)."""
    n = t.shape[-1]
    if t.stride(-1) != 1 and n > 1:
        raise ValueError("last dimension must be contiguous")
    if t.dim() == 1:
        return 1, n
    rows = 1
    for s in t.shape[:-1]:
        rows *= s
    # leading dims must collapse to uniformly strided rows (size-1 dims impose nothing)
    for i in range(t.dim() - 2):
        if t.shape[i] > 1 and t.shape[i + 1] > 1 and t.stride(i) != t.stride(i + 1) * t.shape[i + 1]:
            raise ValueError("leading dimensions must collapse to uniformly strided rows")
    # the row stride is the stride of the innermost leading dim that has more than one entry
    row_stride = next((t.stride(i) for i in range(t.dim() - 2, -1, -1) if t.shape[i] > 1), n)
    return rows, max(row_stride, n)


def set_persistent_sms(n: int) -> None:
    """Cap the persistent GEMM grid of the current CUDA device to n SMs (0 = all)."""
    L.check(L.load().fs_set_persistent_sms(int(n)), "fs_set_persistent_sms")


def set_gemm_pair_mode(on: bool) -> None:
    """Choose the 2-SM (CTA pair) GEMM for M > 128 (default) or always the 1-SM GEMM."""
    L.check(L.load().fs_set_gemm_pair_mode(int(bool(on))), "fs_set_gemm_pair_mode")


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RMSNorm over the last dim (forgeserve/model.py:29-31)."""
    require_cuda(x, w)
    if w.dtype != x.dtype:
        raise TypeError("rmsnorm weight and input must have the same dtype")
    out = torch.empty_like(x, memory_format=torch.contiguous_format) if out is None else out
    rows, xs = _rows(x)
    _, ys = _rows(out)
    lib = L.load()
    L.check(lib.fs_rmsnorm(_p(x), xs, _p(w), _p(out), ys, rows, x.shape[-1], float(eps), dtype_code(x.dtype),
                           _stream(x)), "fs_rmsnorm")
    return out


def linear(x: torch.Tensor, w: torch.Tensor, epilogue: int = L.FS_EPI_STORE, residual: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None, simt: bool = False) -> torch.Tensor:
    """x (..., K) @ w (N, K)^T with a fused epilogue (see fs_gemm). Returns (..., n_out)."""
    require_cuda(x, w, residual, out)
    if w.dtype != x.dtype or (residual is not None and residual.dtype != x.dtype):
        raise TypeError("linear: all operands must share one dtype")
    if w.dim() != 2 or w.stride(1) != 1:
        raise ValueError("linear: weight must be 2-D with contiguous rows")
    K = x.shape[-1]
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"linear: weight has {w.shape[1]} input features, input has {K}")
    n_out = N // 2 if epilogue == L.FS_EPI_SWIGLU else N
    if out is None:
        out = torch.empty(*x.shape[:-1], n_out, dtype=x.dtype, device=x.device)
    M, lda = _rows(x)
    _, ldc = _rows(out)
    ldr = _rows(residual)[1] if residual is not None else 0
    fn = L.load().fs_gemm_simt if simt else L.load().fs_gemm
    ev = gemm_events
    if ev is not None:
        st = torch.cuda.current_stream(x.device)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record(st)
    L.check(fn(_p(x), lda, _p(w), w.stride(0), _p(out), ldc, _p(residual), ldr, M, N, K, n_out, epilogue,
               dtype_code(x.dtype), _stream(x)), "fs_gemm")
    if ev is not None:
        e1.record(st)
        ev.append((e0, e1, 2.0 * M * N * K))
    return out


def linear_to(x: torch.Tensor, w: torch.Tensor, c_ptr: int, ldc: int, system_fence: bool = False) -> None:
    """x (..., K) @ w (N, K)^T stored at device address c_ptr, rows of ldc elements apart (no residual, no
    SwiGLU). c_ptr may be another GPU's buffer mapped with ipc_open; system_fence=True then makes the kernel end
    with a system-scope fence, so its stores are performed by the time the kernel completes."""
    require_cuda(x, w)
    if w.dtype != x.dtype or w.dim() != 2 or w.stride(1) != 1 or w.shape[1] != x.shape[-1]:
        raise ValueError("linear_to: weight must be (N, K) with contiguous rows, in the input's dtype")
    M, lda = _rows(x)
    N, K = w.shape
    if ldc < N:
        raise ValueError("linear_to: output row stride smaller than N")
    epi = L.FS_EPI_STORE | (L.FS_EPI_SYSTEM_FENCE if system_fence else 0)
    ev = gemm_events
    if ev is not None:
        st = torch.cuda.current_stream(x.device)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record(st)
    L.check(L.load().fs_gemm(_p(x), lda, _p(w), w.stride(0), ctypes.c_void_p(c_ptr), ldc, None, 0, M, N, K, N, epi,
                             dtype_code(x.dtype), _stream(x)), "fs_gemm")
    if ev is not None:
        e1.record(st)
        ev.append((e0, e1, 2.0 * M * N * K))


def ipc_handle(t: torch.Tensor) -> bytes:
    """CUDA IPC handle of the allocation holding t, followed by t's byte offset in it (8 bytes, little-endian)."""
    require_cuda(t)
    h = (ctypes.c_char * L.FS_IPC_HANDLE_BYTES)()
    off = ctypes.c_int64()
    L.check(L.load().fs_ipc_handle(_p(t), h, ctypes.byref(off)), "fs_ipc_handle")
    return bytes(h) + int(off.value).to_bytes(8, "little", signed=True)


def ipc_open(handle: bytes) -> int:
    """Map another process's allocation (the first FS_IPC_HANDLE_BYTES bytes of an ipc_handle); returns its base."""
    base = ctypes.c_void_p()
    L.check(L.load().fs_ipc_open(handle[: L.FS_IPC_HANDLE_BYTES], ctypes.byref(base)), "fs_ipc_open")
    return int(base.value)


def copy_2d_to(dst_ptr: int, dpitch: int, src: torch.Tensor) -> None:
    """Copy the rows of a 2-D view `src` (last dim contiguous) to device address dst_ptr, rows dpitch bytes apart,
    on the current stream by the copy engine (dst_ptr may be another GPU's buffer mapped with ipc_open)."""
    require_cuda(src)
    rows, ld = _rows(src)
    width = src.shape[-1] * src.element_size()
    L.check(L.load().fs_copy_2d(ctypes.c_void_p(dst_ptr), int(dpitch), _p(src), ld * src.element_size(), width, rows,
                                _stream(src)), "fs_copy_2d")


def ipc_close(base: int) -> None:
    L.check(L.load().fs_ipc_close(ctypes.c_void_p(base)), "fs_ipc_close")


def rope_kv_write(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                  kv: L.KVCacheDesc, B: int, T: int, nh: int, nkv: int, hd: int, slot_base: int, slot_from_pos: bool,
                  apply_rope: bool = True) -> None:
    require_cuda(qkv, cos, sin, positions)
    rows, ld = _rows(qkv)
    L.check(L.load().fs_rope_kv_write(_p(qkv), ld, _p(cos), _p(sin), cos.shape[0], _p(positions), ctypes.byref(kv), B,
                                      T, nh, nkv, hd, slot_base, int(slot_from_pos), int(apply_rope),
                                      dtype_code(qkv.dtype), _stream(qkv)), "fs_rope_kv_write")


def attention(q: torch.Tensor, kv: L.KVCacheDesc, n_slots: int, positions: torch.Tensor, out: torch.Tensor, B: int,
              T: int, nh: int, nkv: int, hd: int, impl: int = L.FS_ATTN_AUTO) -> torch.Tensor:
    """GQA attention over a cache; impl selects the kernel (FS_ATTN_*), automatic by default."""
    require_cuda(q, positions, out)
    _, ldq = _rows(q)
    _, ldo = _rows(out)
    L.check(L.load().fs_attention_impl(_p(q), ldq, ctypes.byref(kv), n_slots, _p(positions), _p(out), ldo, B, T, nh,
                                       nkv, hd, 1.0 / math.sqrt(hd), int(impl), dtype_code(q.dtype), _stream(q)),
            "fs_attention")
    return out


_DECODE_WS = {}
_DECODE_WS_RETIRED: List[torch.Tensor] = []


def decode_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """A scratch buffer for split decode attention per (device, current stream), grown on demand and reused by the
    calls on that stream (which run one after another). A buffer that is outgrown stays allocated: a CUDA graph
    captured earlier may still address it."""
    key = (str(device), torch.cuda.current_stream(device).cuda_stream)
    ws = _DECODE_WS.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _DECODE_WS_RETIRED.append(ws)
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _DECODE_WS[key] = ws
    return ws


def attention_decode(q: torch.Tensor, kv: L.KVCacheDesc, n_slots: int, positions: torch.Tensor, out: torch.Tensor,
                     B: int, nh: int, nkv: int, hd: int) -> torch.Tensor:
    """Split-KV decode attention: one query per row (positions (B,) or (B, 1))."""
    require_cuda(q, positions, out)
    _, ldq = _rows(q)
    _, ldo = _rows(out)
    lib = L.load()
    need = int(lib.fs_attention_decode_workspace(B, nh, nkv, hd, n_slots))
    ws = decode_workspace(q.device, need) if need > 0 else None
    L.check(lib.fs_attention_decode(_p(q), ldq, ctypes.byref(kv), n_slots, _p(positions), _p(out), ldo, B, nh, nkv, hd,
                                    1.0 / math.sqrt(hd), _p(ws), 0 if ws is None else ws.numel(),
                                    dtype_code(q.dtype), _stream(q)), "fs_attention_decode")
    return out


def kv_store(k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, kv: L.KVCacheDesc) -> None:
    require_cuda(k, v, positions)
    B, nkv, T, hd = k.shape
    k, v = k.contiguous(), v.contiguous()
    L.check(L.load().fs_kv_store(_p(k), _p(v), _p(positions), ctypes.byref(kv), B, T, nkv, hd, dtype_code(k.dtype),
                                 _stream(k)), "fs_kv_store")


def paged_gather(pool: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """pool (num_blocks, nkv, bs, hd), table (B, nb) int64 -> (B, nkv, nb*bs, hd)."""
    require_cuda(pool, table)
    nblk, nkv, bs, hd = pool.shape
    B, nb = table.shape
    out = torch.empty(B, nkv, nb * bs, hd, dtype=pool.dtype, device=pool.device)
    L.check(L.load().fs_paged_gather(_p(pool), _p(table), B, nb, nblk, nkv, bs, hd, _p(out), dtype_code(pool.dtype),
                                     _stream(pool)), "fs_paged_gather")
    return out


def _row_view(t: torch.Tensor, rows: int, cols: int, name: str) -> int:
    """Row stride of t seen as `rows` rows of `cols` values; refuses other sizes and rows that overlap."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2 and shape[0] == rows and shape[1] == cols and stride[1] == 1 and stride[0] >= cols:
        return stride[0]
    n, ld = _rows(t)
    if n != rows or shape[-1] != cols:
        raise ValueError(f"{name} must hold {rows} rows of {cols} values, not {tuple(shape)}")
    if n > 1 and next(stride[i] for i in range(t.dim() - 2, -1, -1) if shape[i] > 1) < cols:
        raise ValueError(f"the rows of {name} overlap")
    return ld


def _check_positions(positions: torch.Tensor, n: int) -> None:
    if positions.dtype != torch.int64 or not positions.is_contiguous() or positions.numel() != n:
        raise ValueError(f"positions must be {n} contiguous int64 values")


def _on_device(device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            require_cuda(t)
            raise RuntimeError(f"tensors on two devices: {device} and {t.device}")


def _check_cache(kv, B: int, nkv: int, hd: int, device: torch.device, dtype: torch.dtype) -> None:
    """The tensors behind a descriptor against a call's sizes (descriptors filled by hand carry none)."""
    keep = getattr(kv, "keep", None)
    if keep is None:
        return
    k, v, table = keep[0], keep[1], keep[2]
    if k.device != device or v.device != device or table.device != device:
        _on_device(device, k, v, table)
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"the cache holds {k.dtype}, the call needs {dtype}")
    shape = k.shape
    if shape[1] != nkv or shape[3] != hd or shape != v.shape:
        raise ValueError(f"the cache holds {shape[1]} heads of {shape[3]}, the call has {nkv} of {hd}")
    if table.dim() > 2 or table.dtype != torch.int64 or table.stride(-1) != 1 and table.shape[-1] > 1:
        raise ValueError("the block table must be int64 with contiguous rows")
    if table.shape[0] < B:
        raise ValueError(f"the block table has {table.shape[0]} rows, the call {B}")


def _check_quant_cache(kv: L.KVQuantDesc, B: int, nkv: int, hd: int, device: torch.device) -> None:
    """A quant_paged_desc against a call's sizes (its tensors were checked against each other when it was made)."""
    about = getattr(kv, "about", None)
    if about is not None and (about[0] != device or about[1] != nkv or about[2] != hd or about[3] < B):
        _on_device(device, kv.keep[0])
        raise ValueError(f"the cache holds {about[1]} heads of {about[2]} for {about[3]} rows, the call has {nkv} of "
                         f"{hd} for {B}")


def _run(what: str, fn, device: torch.device, *args) -> None:
    """fn(*args, stream) on the tensors' device and its current stream; raises on an error status."""
    index = device.index
    if torch.cuda.current_device() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        L.check(status, what)


_ROPE_LAYOUTS = {"half": 0, "interleaved": 1}


def rotary_kv_write(qkv: torch.Tensor, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
                    positions: torch.Tensor, kv, B: int, T: int, nh: int, nkv: int, hd: int, slot_base: int = 0,
                    slot_from_pos: bool = True, layout: str = "half",
                    q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate q and k of the fused q/k/v rows (B*T, (nh + 2 nkv) * hd) and store k and v into the cache.

    cos, sin: fp32 (positions, r/2); the first r values of each head turn, in pairs (x[i], x[i + r/2]) (layout "half")
    or (x[2i], x[2i+1]) ("interleaved"); None rotates nothing. fp32 arithmetic with one rounding, where rope_kv_write
    keeps the reference's bf16 roundings. kv: paged_desc / contiguous_desc (a cache in qkv's dtype) or
    quant_paged_desc (an 8-bit cache). Returns the rotated q: q_out (B*T, nh * hd), or q's place in qkv, rotated in
    place. A negative position marks padding: its q_out row and the cache stay as they were. Two tokens of a call must
    not share a slot."""
    if not qkv.is_cuda:
        require_cuda(qkv)
    dev, M = qkv.device, B * T
    ld = _row_view(qkv, M, (nh + 2 * nkv) * hd, "qkv")
    code = dtype_code(qkv.dtype)
    if layout not in _ROPE_LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved', not {layout!r}")
    _check_positions(positions, M)
    _on_device(dev, positions, cos, sin, q_out)
    rows = rd = cos_p = sin_p = 0
    if cos is not None or sin is not None:
        if (cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32
                or sin.dtype != torch.float32 or not cos.is_contiguous() or not sin.is_contiguous()):
            raise ValueError("cos and sin must be contiguous fp32 tables of one shape (positions, rotary_dim / 2)")
        rows, rd = cos.shape
        rd, cos_p, sin_p = 2 * rd, cos.data_ptr(), sin.data_ptr()
    if q_out is None:
        q_out = (qkv if qkv.dim() == 2 else qkv.view(M, -1))[:, : nh * hd]
        ldq = ld
    else:
        if q_out.dtype != qkv.dtype:
            raise TypeError("q_out must have qkv's dtype")
        ldq = _row_view(q_out, M, nh * hd, "q_out") if nh else 0
    quant = isinstance(kv, L.KVQuantDesc)
    if quant:
        _check_quant_cache(kv, B, nkv, hd, dev)
    else:
        _check_cache(kv, B, nkv, hd, dev, qkv.dtype)
    lib = L.load()
    _run("fs_rotary_kv_write", lib.fs_rotary_kv_write_quant if quant else lib.fs_rotary_kv_write, dev,
         qkv.data_ptr(), ld, q_out.data_ptr(), ldq, cos_p, sin_p, rows, rd, _ROPE_LAYOUTS[layout], positions.data_ptr(),
         kv, B, T, nh, nkv, hd, slot_base, slot_from_pos, code)
    return q_out


def kv_dequant(kv: L.KVQuantDesc, B: int, n_slots: int, nkv: int, hd: int, dtype: torch.dtype,
               positions: Optional[torch.Tensor] = None):
    """The first n_slots slots of every row of an 8-bit cache as dense (k, v), each (B, nkv, n_slots, hd) of dtype. A block
    number outside the cache reads as zeros and raises the bad slot flag; with positions (B, T), those of the queries that
    look at the result, only where a row's last one reaches the block."""
    codes = kv.keep[0]
    if not codes.is_cuda:
        require_cuda(codes)
    dev = codes.device
    code = dtype_code(dtype)
    _check_quant_cache(kv, B, nkv, hd, dev)
    k = torch.empty((B, nkv, n_slots, hd), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if positions is None:
        _run("fs_kv_dequant", L.load().fs_kv_dequant, dev, kv, B, n_slots, nkv, hd, k.data_ptr(), v.data_ptr(), code)
    elif positions.numel():
        T = positions.shape[-1]
        _check_positions(positions, B * T)
        _on_device(dev, positions)
        _run("fs_kv_dequant_for", L.load().fs_kv_dequant_for, dev, kv, B, n_slots, nkv, hd, positions.data_ptr(), T,
             k.data_ptr(), v.data_ptr(), code)
    else:
        raise ValueError("kv_dequant: positions of at least one query a row needed")
    return k, v


def attention_decode_quant(q: torch.Tensor, kv: L.KVQuantDesc, n_slots: int, positions: torch.Tensor,
                           out: torch.Tensor, B: int, nh: int, nkv: int, hd: int) -> torch.Tensor:
    """attention_decode over an 8-bit cache: one query per row (positions (B,) or (B, 1)), any n_heads / n_kv_heads,
    even head_dim up to 256. A row with a negative position sees no slot and gets zeros."""
    if not q.is_cuda:
        require_cuda(q)
    dev = q.device
    _on_device(dev, positions, out)
    if out.dtype != q.dtype:
        raise TypeError("attention_decode_quant: out must have q's dtype")
    code = dtype_code(q.dtype)
    ldq, ldo = _row_view(q, B, nh * hd, "q"), _row_view(out, B, nh * hd, "out")
    _check_positions(positions, B)
    _check_quant_cache(kv, B, nkv, hd, dev)
    lib = L.load()
    # Allocated by each call: the allocator hands it out in stream order, and a captured call's stays with its graph.
    need = lib.fs_attention_decode_quant_workspace(B, nh, nkv, hd, n_slots)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _run("fs_attention_decode_quant", lib.fs_attention_decode_quant, dev, q.data_ptr(), ldq, kv, n_slots,
         positions.data_ptr(), out.data_ptr(), ldo, B, nh, nkv, hd, 1.0 / math.sqrt(hd),
         0 if ws is None else ws.data_ptr(), need, code)
    return out


def embed(ids: torch.Tensor, table: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """table[ids] for int64 ids on the table's device (nn.Embedding)."""
    require_cuda(ids, table)
    ids = ids.contiguous()
    if ids.dtype != torch.int64:
        ids = ids.long()
    V, d = table.shape
    if out is None:
        out = torch.empty(*ids.shape, d, dtype=table.dtype, device=table.device)
    L.check(L.load().fs_embed(_p(ids), ids.numel(), _p(table), V, d, _p(out), dtype_code(table.dtype), _stream(table)),
            "fs_embed")
    return out


def argmax(x: torch.Tensor) -> torch.Tensor:
    """argmax over the last dim (lowest index on ties), int64 result of shape x.shape[:-1]."""
    require_cuda(x)
    rows, rs = _rows(x)
    out = torch.empty(x.shape[:-1], dtype=torch.int64, device=x.device)
    L.check(L.load().fs_argmax(_p(x), rows, x.shape[-1], rs, _p(out), dtype_code(x.dtype), _stream(x)), "fs_argmax")
    return out


def contiguous_desc(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor) -> L.KVCacheDesc:
    """Descriptor of a per-row cache k, v of shape (B, nkv, capacity, hd) (contiguous); table = arange(B)."""
    B, nkv, cap, hd = k.shape
    desc = L.KVCacheDesc(k.data_ptr(), v.data_ptr(), table.data_ptr(), 1, 1, cap, nkv * cap * hd, cap * hd, B)
    desc.keep = (k, v, table)          # the descriptor holds raw pointers: keep the tensors alive with it
    return desc


def paged_desc(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor) -> L.KVCacheDesc:
    """Descriptor of a paged pool k, v of shape (num_blocks, nkv, block_size, hd); table (B, nb) int64."""
    nblk, nkv, bs, hd = k.shape
    desc = L.KVCacheDesc(k.data_ptr(), v.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1], bs,
                         nkv * bs * hd, bs * hd, nblk)
    desc.keep = (k, v, table)
    return desc


def _strides(t: torch.Tensor) -> tuple:
    """t's strides, those of dimensions of one entry (which address nothing) as if t were contiguous from there on."""
    out, step = [], 1
    for n, st in zip(reversed(t.shape), reversed(t.stride())):
        out.append(step if n == 1 else st)
        step *= n
    return tuple(reversed(out))


_PACK_QUANT = struct.Struct("13q").pack   # the fields of KVQuantDesc, all 8 bytes


def quant_paged_desc(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                     table: torch.Tensor) -> L.KVQuantDesc:
    """Descriptor of an 8-bit paged pool: codes k, v float8_e4m3fn (num_blocks, nkv, block_size, hd), scales fp32
    (num_blocks, nkv, block_size); table (B, nb) int64."""
    if k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
        raise TypeError("quant_paged_desc: k and v must be float8_e4m3fn")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise TypeError("quant_paged_desc: the scales must be float32")
    if k.dim() != 4 or table.dim() != 2:
        raise ValueError("quant_paged_desc: k and v must be 4-D, the block table 2-D")
    nblk, nkv, bs, hd = shape = k.shape
    rows = (nblk, nkv, bs)
    if v.shape != shape or k_scale.shape != rows or v_scale.shape != rows:
        raise ValueError("quant_paged_desc: k, v and their scales must describe one pool")
    strides, cols = k.stride(), k_scale.stride()
    if v.stride() != strides or v_scale.stride() != cols or strides[2:] != (hd, 1) or cols[2] != 1:
        strides, cols = _strides(k), _strides(k_scale)   # apart from the dimensions of one entry
        if _strides(v) != strides or _strides(v_scale) != cols or strides[2:] != (hd, 1) or cols[2] != 1:
            raise ValueError("quant_paged_desc: the slots of a (block, head) must lie contiguously, k and v alike")
    s0, s1, _, _ = strides
    c0, c1, _ = cols
    (n, width), (t0, t1) = table.shape, table.stride()
    if table.dtype != torch.int64 or t1 != 1 and width > 1:
        raise ValueError("the block table must be int64 with contiguous rows")
    dev = k.device
    if v.device != dev or k_scale.device != dev or v_scale.device != dev or table.device != dev:
        _on_device(dev, v, k_scale, v_scale, table)
    desc = L.KVQuantDesc.from_buffer_copy(_PACK_QUANT(
        k.data_ptr(), v.data_ptr(), table.data_ptr(), t0, width, bs, s0, s1, nblk, k_scale.data_ptr(),
        v_scale.data_ptr(), c0, c1))
    desc.keep = (k, v, table, k_scale, v_scale)
    desc.about = (dev, nkv, hd, n)
    return desc
