"""Python-side handles over the C ABI, for torch (ROCm) device tensors.

PyTorch is used only for device memory and streams: every computation runs in
libcx_moe.so.  Calls are enqueued on torch's current stream of the tensors'
device.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Sequence, Union

import numpy as np
import torch

from ._lib import (BF16, E4M3, F32, FP16, CxError, DeviceInfo, ExpertDesc, MoeLayerRequestInfo,
                   Q4Desc, check, lib)

_TORCH_TO_CX = {torch.float16: FP16, torch.bfloat16: BF16, torch.float32: F32}
_CX_TO_TORCH = {FP16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}


def cx_dtype(t: torch.dtype) -> int:
    try:
        return _TORCH_TO_CX[t]
    except KeyError:
        raise TypeError(f"unsupported dtype {t}") from None


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _rows_2d(t: torch.Tensor) -> tuple[int, int]:
    if t.dim() != 2:
        raise ValueError(f"expected a 2D tensor, got shape {tuple(t.shape)}")
    return t.shape[0], t.shape[1]


def _places(place: torch.Tensor, n_tokens: int) -> int:
    if place.dtype != torch.int32 or place.dim() != 2 or place.shape[0] != n_tokens or not place.is_contiguous():
        raise ValueError(f"place must be contiguous int32 [{n_tokens}, top_k]")
    return place.shape[1]


def _check_pairs(rows: int, n_tokens: int, top_k: int, weights: Optional[torch.Tensor]) -> None:
    if rows != n_tokens * top_k:
        raise ValueError(f"{rows} sorted rows, {n_tokens} x {top_k} pairs")
    if weights is not None and (weights.shape != (n_tokens, top_k) or weights.dtype != torch.float32):
        raise ValueError(f"weights must be fp32 [{n_tokens}, {top_k}]")


def _device(index: int) -> torch.device:
    return torch.device("cuda", index)


def _outside_autograd(name: str, gradient: str, *tensors: Optional[torch.Tensor]) -> None:
    """A result without a graph must not pass for one with it."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name} records no graph: call it under torch.no_grad() or in an autograd.Function "
                         f"whose backward is {gradient}")


def _stream(device: int) -> int:
    """The current stream's handle; without a Stream object around it, where torch has
    that (a microsecond less a call).  Looked up by the call: the module also serves programs
    whose torch has no GPU build."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return torch.cuda.current_stream(device).cuda_stream if raw is None else raw(device)


def device_count() -> int:
    n = C.c_int(0)
    check(lib().cx_device_count(C.byref(n)))
    return n.value


def device_info(device: int = 0) -> dict:
    info = DeviceInfo()
    check(lib().cx_device_query(device, C.byref(info)))
    return {
        "name": info.name.decode(), "arch": info.arch.decode(),
        "total_mem_bytes": info.total_mem_bytes, "free_mem_bytes": info.free_mem_bytes,
        "capability_flags": info.capability_flags, "compute_units": info.compute_units,
        "num_xcds": info.num_xcds,
    }


def arena_stats(device: int = 0) -> tuple[int, int]:
    u, r = C.c_uint64(0), C.c_uint64(0)
    check(lib().cx_arena_stats(device, C.byref(u), C.byref(r)))
    return u.value, r.value


LAYOUT_ROWS, LAYOUT_TILE16 = 0, 1  # cx_expert_desc::gu_layout


def untile16(a: np.ndarray) -> np.ndarray:
    """CX_LAYOUT_TILE16 bytes of a [rows, cols] matrix (as read back from the
    device, in a [rows, cols] array) in row-major order: tiles of 16 rows x
    128 columns in row-group, then column order; inside a tile, the 32 bytes
    of row r, columns 32q .. 32q + 31 at (16q + r) * 32."""
    rows, cols = a.shape
    t = a.reshape(rows // 16, cols // 128, 4, 16, 32)   # [row group][k-block][quarter][row][32 B]
    return np.ascontiguousarray(t.transpose(0, 3, 1, 2, 4)).reshape(rows, cols)


def tile16(a: np.ndarray) -> np.ndarray:
    """Row-major [rows, cols] bytes in CX_LAYOUT_TILE16 order (untile16's inverse)."""
    rows, cols = a.shape
    t = np.ascontiguousarray(a).reshape(rows // 16, 16, cols // 128, 4, 32)
    return np.ascontiguousarray(t.transpose(0, 2, 3, 1, 4)).reshape(rows, cols)


class Expert:
    """A device-resident fp8 expert living in the library's HBM arena."""

    def __init__(self, device: int, desc: ExpertDesc):
        self.device = device
        self.desc = desc
        self._live = True

    @classmethod
    def upload(cls, device: int, w_up, s_up, w_gate, s_gate, w_down, s_down, *,
               row_block: int = 128, col_block: int = 128, tiled: Optional[bool] = None) -> "Expert":
        """Upload host fp8 bytes + fp32 scale_inv (the UploadExpertAmdV2 path).
        Up and gate are re-tiled on the device (CX_LAYOUT_TILE16) when the
        shape allows, as the node's upload does; tiled=False keeps them
        row-major."""
        w_up, w_gate, w_down = (np.ascontiguousarray(a, np.uint8) for a in (w_up, w_gate, w_down))
        s_up, s_gate, s_down = (np.ascontiguousarray(a, np.float32) for a in (s_up, s_gate, s_down))
        inter, hidden = w_up.shape
        if w_gate.shape != (inter, hidden) or w_down.shape != (hidden, inter):
            raise ValueError("expert shapes must be up/gate [I,H] and down [H,I]")
        ok = inter % 16 == 0 and hidden % 128 == 0
        if tiled is None:
            tiled = ok
        elif tiled and not ok:
            raise ValueError("tiled gate/up needs inter % 16 == 0 and hidden % 128 == 0")
        ptrs = []
        try:
            for w, s, t in ((w_up, s_up, tiled), (w_gate, s_gate, tiled), (w_down, s_down, False)):
                dw, ds = C.c_void_p(), C.c_void_p()
                up = lib().cx_upload_matrix_tiled if t else lib().cx_upload_matrix
                check(up(device, w.ctypes.data, w.shape[0], w.shape[1], s.ctypes.data, s.size,
                         C.byref(dw), C.byref(ds)))
                ptrs += [dw.value, ds.value]
        except Exception:
            for p in ptrs:
                lib().cx_free_device(device, p)
            raise
        d = ExpertDesc(*ptrs, hidden, inter, row_block, col_block, row_block, col_block,
                       row_block, col_block, LAYOUT_TILE16 if tiled else LAYOUT_ROWS)
        return cls(device, d)

    @classmethod
    def generate(cls, device: int, seed: int, stream_base: int, hidden: int = 7168,
                 inter: int = 2048, block: int = 128, std: float = 0.02) -> "Expert":
        d = ExpertDesc()
        check(lib().cx_gen_expert(device, seed, stream_base, hidden, inter, block, std, C.byref(d)))
        return cls(device, d)

    @property
    def hidden(self) -> int:
        return self.desc.hidden

    @property
    def inter(self) -> int:
        return self.desc.inter

    def download(self) -> dict:
        """Copy the resident bytes back to host numpy arrays (for checks)."""
        H, I = self.hidden, self.inter
        out = {}
        specs = (("w_up", self.desc.w_up, (I, H), np.uint8, self.desc.up_rb, self.desc.up_cb),
                 ("s_up", self.desc.s_up, None, np.float32, self.desc.up_rb, self.desc.up_cb),
                 ("w_gate", self.desc.w_gate, (I, H), np.uint8, self.desc.gate_rb, self.desc.gate_cb),
                 ("s_gate", self.desc.s_gate, None, np.float32, self.desc.gate_rb, self.desc.gate_cb),
                 ("w_down", self.desc.w_down, (H, I), np.uint8, self.desc.down_rb, self.desc.down_cb),
                 ("s_down", self.desc.s_down, None, np.float32, self.desc.down_rb, self.desc.down_cb))
        for name, ptr, shape, dt, rb, cb in specs:
            if shape is None:
                rows, cols = (I, H) if name != "s_down" else (H, I)
                shape = ((rows + rb - 1) // rb, (cols + cb - 1) // cb)
            a = np.empty(shape, dt)
            _hip_d2h(a, ptr)
            if name in ("w_up", "w_gate") and self.desc.gu_layout == LAYOUT_TILE16:
                a = untile16(a)
            out[name] = a
        out.update(hidden=H, inter=I, rb=self.desc.up_rb, cb=self.desc.up_cb)
        return out

    def free(self) -> None:
        if self._live:
            check(lib().cx_free_expert(self.device, C.byref(self.desc)))
            self._live = False


def _hip_d2h(dst: np.ndarray, src_ptr: int) -> None:
    """hipMemcpy device->host through the HIP runtime already loaded by torch."""
    torch.cuda.synchronize()
    hip = C.CDLL("libamdhip64.so")
    hip.hipMemcpy.restype = C.c_int
    hip.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    rc = hip.hipMemcpy(dst.ctypes.data, src_ptr, dst.nbytes, 2)
    if rc != 0:
        raise RuntimeError(f"hipMemcpy D2H failed: {rc}")


class Layer:
    """Device table of resident experts (local ids 0..E-1) + optional shared expert."""

    def __init__(self, ctx: "Context", experts: Sequence[Optional[Expert]],
                 shared: Optional[Expert] = None):
        self.ctx = ctx
        self.n_experts = len(experts)
        self.experts = list(experts)
        self.shared = shared
        arr = (C.POINTER(ExpertDesc) * self.n_experts)()
        for i, e in enumerate(experts):
            arr[i] = C.pointer(e.desc) if e is not None else C.POINTER(ExpertDesc)()
        h = C.c_void_p()
        check(lib().cx_layer_create(ctx.handle, self.n_experts, arr,
                                    C.byref(shared.desc) if shared is not None else None,
                                    C.byref(h)))
        self.handle = h.value
        first = next(e for e in list(experts) + [shared] if e is not None)
        self.hidden, self.inter = first.hidden, first.inter

    def close(self) -> None:
        if self.handle:
            lib().cx_layer_destroy(self.ctx.handle, self.handle)
            self.handle = None


class Norm(NamedTuple):
    """What Context.rms_norm was asked for (None where it was not)."""
    sum: Optional[torch.Tensor]    # x + residual, in x's type
    y: Optional[torch.Tensor]
    q: Optional[torch.Tensor]      # float8_e4m3fn
    scale: Optional[torch.Tensor]  # fp32 [T, ceil(H / 128)]


class Q4Matrix:
    """A stack of matrices with 4-bit weights, packed in the library's HBM arena
    (cx_q4_desc): e2m1 codes and a bf16 scale per row and `group` columns."""

    def __init__(self, device: int, desc: Q4Desc):
        self.device = device
        self.desc = desc
        self._live = True
        self._scratch: dict = {}  # sizes by call shape

    @classmethod
    def pack(cls, codes: torch.Tensor, scales: torch.Tensor, cols: int, *, group: int = 128,
             gated: bool = False) -> "Q4Matrix":
        """codes: uint8 [n_mats, rows, ceil(cols / 2)] (or [rows, ...] for one), two
        columns a byte, the even one in the lower nibble; scales: bf16 [n_mats,
        rows, ceil(cols / group)].  gated: the rows are a gate matrix and then
        an up matrix of the same size, whose product is silu(gate) * up."""
        if codes.dim() == 2:
            codes, scales = codes.unsqueeze(0), scales.unsqueeze(0)
        if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16:
            raise TypeError("codes must be uint8 and scales bfloat16")
        if group not in (32, 64, 128):
            raise ValueError("group must be 32, 64 or 128")
        E, N = codes.shape[:2]
        if codes.dim() != 3 or cols < 1 or codes.shape[2] != (cols + 1) // 2 or \
                scales.shape != (E, N, -(-cols // group)):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold "
                             f"matrices of {cols} columns in groups of {group}")
        if codes.device.type != "cuda" or scales.device != codes.device:
            raise ValueError("codes and scales must be on one HIP device")
        codes, scales = codes.contiguous(), scales.contiguous()
        dev, d = codes.device.index, Q4Desc()
        check(lib().cx_q4_pack(dev, codes.data_ptr(), scales.data_ptr(), E, N, cols, group, int(gated),
                               _stream(dev), C.byref(d)))
        return cls(dev, d)

    @property
    def out_cols(self) -> int:
        """Columns of a product with this matrix."""
        return self.desc.rows // 2 if self.desc.gated else self.desc.rows

    def free(self) -> None:
        if self._live:
            check(lib().cx_q4_free(self.device, C.byref(self.desc)))
            self._live = False


class Q4Layer:
    """A layer of 4-bit experts: `gate_up` a gated stack [E, 2 * inter, hidden],
    `down` a stack [E, hidden, inter], `shared` the shared expert's two (stacks of
    one), if the layer has one.  Context.moe and Context.moe_layer take it in
    place of a Layer, and so does moe_dispatch.LocalNode.

    `experts`: the ids of the layer's experts that the stacks hold, in their order,
    of n_experts in all (one more than the largest); by default 0 .. E - 1.  A route to
    another expert is left out and reported by Context.sync."""

    def __init__(self, ctx: "Context", gate_up: Q4Matrix, down: Q4Matrix,
                 shared: Optional[tuple[Q4Matrix, Q4Matrix]] = None, *,
                 experts: Optional[Sequence[int]] = None, n_experts: Optional[int] = None):
        g, d = gate_up.desc, down.desc
        if not g.gated or d.gated or g.n_mats != d.n_mats or g.rows != 2 * d.cols or g.cols != d.rows:
            raise ValueError("a layer's matrices must be gated [E, 2 * inter, hidden] and [E, hidden, inter]")
        for own, of in zip(shared or (), (g, d)):
            s = own.desc
            if (s.n_mats, s.rows, s.cols, s.group, s.gated) != (1, of.rows, of.cols, of.group, of.gated):
                raise ValueError("the shared expert must have the layer's sizes and groups")
        if any(m.device != ctx.device for m in (gate_up, down, *(shared or ()))):
            raise ValueError("a layer's matrices must be on its context's device")
        self.ctx = ctx
        self.gate_up, self.down, self.shared = gate_up, down, shared
        held = list(range(g.n_mats)) if experts is None else [int(e) for e in experts]
        self.n_experts = max(held) + 1 if n_experts is None and held else n_experts or 0
        if len(held) != g.n_mats or len(set(held)) != len(held) or min(held) < 0 or max(held) >= self.n_experts:
            raise ValueError(f"experts must be {g.n_mats} different ids below n_experts")
        self.hidden, self.inter = d.rows, d.cols
        self.experts = [None] * self.n_experts  # entry i: who holds expert i here
        for e in held:
            self.experts[e] = self
        # slot in the stacks by id + 1: -1 for no route, one past the stacks for an expert that they do not hold
        self._slots = None
        if held != list(range(self.n_experts)):
            slots = [-1] + [g.n_mats] * (self.n_experts + 1)
            for i, e in enumerate(held):
                slots[e + 1] = i
            self._slots = torch.tensor(slots, dtype=torch.int32, device=_device(ctx.device))
        self._scratch: dict = {}  # sizes by tokens and top_k


class Context:
    """One per device and worker thread (cx_ctx)."""

    def __init__(self, device: int = 0):
        self.device = device
        h = C.c_void_p()
        check(lib().cx_ctx_create(device, C.byref(h)))
        self.handle = h.value

    def close(self) -> None:
        if self.handle:
            lib().cx_ctx_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def stream(self) -> int:
        return _stream(self.device)

    def sync(self) -> None:
        check(lib().cx_ctx_sync(self.handle, self.stream()))

    def profile(self, enable: bool) -> None:
        """Start (clearing totals) / stop per-kernel HIP-event timing."""
        check(lib().cx_ctx_profile(self.handle, int(enable)))

    def profile_read(self, kernel: str) -> tuple[int, float]:
        """(launches, summed ms) of one kernel since profiling started."""
        n, ms = C.c_int(0), C.c_double(0.0)
        check(lib().cx_ctx_profile_read(self.handle, kernel.encode(), C.byref(n), C.byref(ms)))
        return n.value, ms.value

    # -- single expert -----------------------------------------------------
    def expert_run(self, expert: Expert, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None,
                   want_f32: bool = False):
        x = x.contiguous()
        T = x.shape[0] if x.dim() == 2 else 1
        out_dtype = out_dtype or x.dtype
        y = torch.empty((T, expert.hidden), dtype=out_dtype, device=x.device)
        yf = torch.empty((T, expert.hidden), dtype=torch.float32, device=x.device) if want_f32 else None
        check(lib().cx_expert_run(self.handle, C.byref(expert.desc), x.data_ptr(), cx_dtype(x.dtype),
                                  T, y.data_ptr(), cx_dtype(out_dtype), _ptr(yf), self.stream()))
        return (y, yf) if want_f32 else y

    def expert_run_host(self, expert: Expert, x_bytes: bytes, in_dtype: int, n_tokens: int,
                        out_dtype: int) -> bytes:
        xb = np.frombuffer(x_bytes, np.uint8)
        out = np.empty(n_tokens * expert.hidden * 2, np.uint8)
        check(lib().cx_expert_run_host(self.handle, C.byref(expert.desc), xb.ctypes.data, xb.size,
                                       in_dtype, n_tokens, out.ctypes.data, out.size, out_dtype))
        return out.tobytes()

    # -- router --------------------------------------------------------------
    def route(self, x: torch.Tensor, w_router: torch.Tensor, bias: torch.Tensor, *,
              resident: Optional[torch.Tensor] = None, n_group: int = 8, topk_group: int = 4,
              top_k: int = 8, norm_topk_prob: bool = True, routed_scaling_factor: float = 2.5):
        x = x.contiguous()
        if x.dim() == 1:
            x = x.unsqueeze(0)
        T, H = x.shape
        E = w_router.shape[0]
        ids = torch.empty((T, top_k), dtype=torch.int32, device=x.device)
        w = torch.empty((T, top_k), dtype=torch.float32, device=x.device)
        check(lib().cx_route(self.handle, x.data_ptr(), cx_dtype(x.dtype),
                             w_router.contiguous().data_ptr(), cx_dtype(w_router.dtype),
                             bias.contiguous().data_ptr(), _ptr(resident), T, H, E, n_group,
                             topk_group, top_k, int(norm_topk_prob), routed_scaling_factor,
                             ids.data_ptr(), w.data_ptr(), self.stream()))
        return ids, w

    def route_logits(self, n_tokens: int, n_experts: int, device) -> torch.Tensor:
        """fp64 router logits [n_tokens, n_experts] of the last route call."""
        out = torch.empty((n_tokens, n_experts), dtype=torch.float64, device=device)
        check(lib().cx_route_logits(self.handle, out.data_ptr(), n_tokens, n_experts,
                                    self.stream()))
        return out

    # -- rows around the experts -------------------------------------------------
    def _here(self, *tensors: Optional[torch.Tensor]) -> None:
        for t in tensors:
            if t is not None and t.get_device() != self.device:  # -1 on the CPU
                raise ValueError(f"tensor on {t.device}, context on cuda:{self.device}")

    def rms_norm(self, x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                 residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                 want_y: bool = True, quantize: bool = False) -> Norm:
        """RMS norm of x (+ residual) [T, H]: `sum` the residual stream where a
        residual is given, `y` in out_dtype (x's), and with quantize `q` in e4m3
        with `scale` per token and 128 columns."""
        self._here(x, weight, residual)
        T, H = _rows_2d(x)
        if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
            raise ValueError("residual must have x's shape and type")
        if weight is not None and weight.shape != (H,):
            raise ValueError(f"weight must be [{H}]")
        if not (want_y or quantize):
            raise ValueError("nothing to compute: want_y or quantize")
        x = x.contiguous()
        residual = None if residual is None else residual.contiguous()
        weight = None if weight is None else weight.contiguous()
        dt = cx_dtype(x.dtype)
        out_dtype = out_dtype or x.dtype
        s = None if residual is None else torch.empty_like(x)
        y = torch.empty_like(x, dtype=out_dtype) if want_y else None
        q = scale = None
        if quantize:
            q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
            scale = x.new_empty((T, (H + 127) // 128), dtype=torch.float32)
        check(lib().cx_rms_norm(self.handle, x.data_ptr(), dt, _ptr(residual), _ptr(weight),
                                dt if weight is None else cx_dtype(weight.dtype), T, H, eps, _ptr(s), _ptr(y),
                                cx_dtype(out_dtype), _ptr(q), _ptr(scale), self.stream()))
        return Norm(s, y, q, scale)

    def sort_tokens(self, ids: torch.Tensor, n_experts: int):
        """(order [T * K], offsets [n_experts + 1], place [T, K]), all int32: the
        pairs t * K + k sorted by expert (cx_sort_tokens).  ids: any integer type."""
        self._here(ids)
        T, K = _rows_2d(ids)
        if ids.dtype == torch.bool or ids.is_floating_point() or ids.is_complex():
            raise TypeError(f"ids must be integers, not {ids.dtype}")
        if ids.element_size() >= 4 and ids.dtype != torch.int32:  # what does not fit 32 bits names no expert, and must not become one that does
            ids = ids.to(torch.int64).clamp(-1, 2 ** 31 - 1)
        ids = ids.to(torch.int32).contiguous()
        order = torch.empty(T * K, dtype=torch.int32, device=ids.device)
        offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=ids.device)
        place = torch.empty((T, K), dtype=torch.int32, device=ids.device)
        check(lib().cx_sort_tokens(self.handle, ids.data_ptr(), T, K, n_experts, order.data_ptr(),
                                   offsets.data_ptr(), place.data_ptr(), self.stream()))
        return order, offsets, place

    def gather_rows(self, x: torch.Tensor, place: torch.Tensor) -> torch.Tensor:
        """Rows of x [T, H] (any type) in sorted order [T * K, H]; zeros where a
        pair has no expert.  Its gradient: combine_rows(dxs, place), by the caller's
        autograd.Function (tensors that require grad are refused outside of one)."""
        self._here(x, place)
        _outside_autograd("gather_rows", "combine_rows(dxs, place)", x)
        T, H = _rows_2d(x)
        K = _places(place, T)
        x = x.contiguous()
        xs = torch.empty((T * K, H), dtype=x.dtype, device=x.device)
        check(lib().cx_gather_rows(self.handle, x.data_ptr(), H * x.element_size(), place.data_ptr(), T, K,
                                   xs.data_ptr(), self.stream()))
        return xs

    def combine_rows(self, ys: torch.Tensor, place: torch.Tensor, weights: Optional[torch.Tensor] = None, *,
                     add: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """Sorted rows ys [T * K, H] back to tokens: [T, H] in out_dtype (ys's),
        the sum over k of weights[t, k] * ys[place[t, k]] (+ add[t]).  Its gradient:
        combine_rows_grad, by the caller's autograd.Function (as gather_rows)."""
        self._here(ys, place, weights, add)
        _outside_autograd("combine_rows", "combine_rows_grad", ys, weights, add)
        P, H = _rows_2d(ys)
        T = place.shape[0]
        K = _places(place, T)
        out_dtype = out_dtype or ys.dtype
        _check_pairs(P, T, K, weights)
        if add is not None and (add.shape != (T, H) or add.dtype != out_dtype):
            raise ValueError(f"add must be [{T}, {H}] in the output's type")
        ys = ys.contiguous()
        weights = None if weights is None else weights.contiguous()
        add = None if add is None else add.contiguous()
        out = torch.empty((T, H), dtype=out_dtype, device=ys.device)
        check(lib().cx_combine_rows(self.handle, ys.data_ptr(), cx_dtype(ys.dtype), place.data_ptr(),
                                    _ptr(weights), _ptr(add), T, K, H, out.data_ptr(), cx_dtype(out_dtype),
                                    None, self.stream()))
        return out

    def combine_rows_grad(self, dout: torch.Tensor, ys: torch.Tensor, place: torch.Tensor,
                          weights: Optional[torch.Tensor] = None):
        """(dys [T * K, H] in ys's type, dw fp32 [T, K]) of combine_rows."""
        self._here(dout, ys, place, weights)
        P, H = _rows_2d(ys)
        T = place.shape[0]
        K = _places(place, T)
        _check_pairs(P, T, K, weights)
        if dout.shape != (T, H):
            raise ValueError(f"dout must be [{T}, {H}]")
        dout, ys = dout.contiguous(), ys.contiguous()
        weights = None if weights is None else weights.contiguous()
        dys = torch.empty_like(ys)
        dw = torch.empty((T, K), dtype=torch.float32, device=ys.device)
        check(lib().cx_combine_rows_grad(self.handle, dout.data_ptr(), cx_dtype(dout.dtype), ys.data_ptr(),
                                         cx_dtype(ys.dtype), place.data_ptr(), _ptr(weights), T, K, H,
                                         dys.data_ptr(), dw.data_ptr(), self.stream()))
        return dys, dw

    # -- 4-bit weights -------------------------------------------------------------
    def q4_matmul(self, w: Q4Matrix, x: torch.Tensor, *, x_scale: Optional[torch.Tensor] = None,
                  offsets: Optional[torch.Tensor] = None, order: Optional[torch.Tensor] = None,
                  top_k: int = 1, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """x W^T (silu(x G^T) * (x U^T) for a gated matrix) in out_dtype (x's; bf16
        for e4m3 x, which comes with rms_norm's scale).  A stack of matrices takes
        the rows offsets[e] .. offsets[e + 1] - 1 through matrix e; with `order`,
        row p is row order[p] // top_k of x (sort_tokens' offsets and order)."""
        self._here(x, x_scale, offsets, order)
        T, K = _rows_2d(x)
        d = w.desc
        if w.device != self.device:
            raise ValueError(f"matrix on cuda:{w.device}, context on cuda:{self.device}")
        if not w._live:
            raise ValueError("the matrix has been freed")
        if K != d.cols:
            raise ValueError(f"x has {K} columns, the matrix {d.cols}")
        f8 = x.dtype == torch.float8_e4m3fn
        if f8 != (x_scale is not None):
            raise ValueError("x_scale comes with e4m3 x, and only with it")
        if f8 and (x_scale.shape != (T, (K + 127) // 128) or x_scale.dtype != torch.float32):
            raise ValueError(f"x_scale must be fp32 [{T}, {(K + 127) // 128}]")
        for name, t, n in (("offsets", offsets, d.n_mats + 1), ("order", order, None)) if offsets is not None or \
                order is not None else ():
            if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous()
                                  or (n is not None and t.shape[0] != n)):
                raise ValueError(f"{name} must be a contiguous int32 vector" + (f" of {n}" if n else ""))
        P = T if order is None else order.shape[0]
        x = x.contiguous()
        x_scale = None if x_scale is None else x_scale.contiguous()
        out_dtype = out_dtype or (torch.bfloat16 if f8 else x.dtype)
        y = torch.empty((P, w.out_cols), dtype=out_dtype, device=x.device)
        dt = E4M3 if f8 else cx_dtype(x.dtype)
        key = (dt, T, P, offsets is None)
        size = w._scratch.get(key)
        if size is None:
            size = w._scratch[key] = lib().cx_q4_scratch(C.byref(d), dt, T, P, int(offsets is not None))
        scratch = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        check(lib().cx_q4_matmul(self.handle, C.byref(d), x.data_ptr(), dt,
                                 _ptr(x_scale), T, _ptr(order), top_k, _ptr(offsets), P, y.data_ptr(),
                                 cx_dtype(out_dtype), _ptr(scratch), size, self.stream()))
        return y

    def _q4_ready(self, layer: Q4Layer, x: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
        """What a call on a 4-bit layer needs of it and of x, before anything is launched."""
        self._here(x, *others)
        if layer.gate_up.device != self.device:
            raise ValueError(f"layer on cuda:{layer.gate_up.device}, context on cuda:{self.device}")
        if not all(m._live for m in (layer.gate_up, layer.down, *(layer.shared or ()))):
            raise ValueError("a matrix of the layer has been freed")
        if x.dim() != 2 or x.shape[1] != layer.hidden:
            raise ValueError(f"x has {x.shape[-1] if x.dim() else 0} columns in {x.dim()} dimensions, the layer {layer.hidden} in 2")

    def _q4_moe(self, layer: Q4Layer, x, topk_ids, topk_w, y, yf):
        self._q4_ready(layer, x, topk_ids, topk_w)
        T, K = x.shape[0], topk_ids.shape[1] if topk_ids.dim() == 2 else -1
        if topk_ids.shape != (T, K) or topk_w.shape != (T, K):
            raise ValueError(f"routes must be [{T}, top_k]")
        if layer._slots is not None:
            topk_ids = layer._slots[topk_ids.clamp(-1, layer.n_experts).long() + 1]
        gu, dn = C.byref(layer.gate_up.desc), C.byref(layer.down.desc)
        sg, sd = (C.byref(m.desc) for m in layer.shared) if layer.shared else (None, None)
        size = layer._scratch.get((T, K))
        if size is None:
            size = layer._scratch[T, K] = lib().cx_q4_moe_scratch(gu, dn, int(layer.shared is not None), T, K)
        scratch = torch.empty(size, dtype=torch.uint8, device=x.device)
        check(lib().cx_q4_moe(self.handle, gu, dn, sg, sd, x.data_ptr(), cx_dtype(x.dtype), T,
                              topk_ids.data_ptr(), topk_w.data_ptr(), K, y.data_ptr(), cx_dtype(y.dtype),
                              _ptr(yf), scratch.data_ptr(), size, self.stream()))

    # -- grouped MoE -----------------------------------------------------------
    def moe(self, layer: Union[Layer, Q4Layer], x: torch.Tensor, topk_ids: torch.Tensor, topk_w: torch.Tensor, *,
            out_dtype: Optional[torch.dtype] = None, want_f32: bool = False,
            prefill: Optional[bool] = None):
        x = x.contiguous()
        T = x.shape[0]
        K = topk_ids.shape[1] if topk_ids.dim() == 2 else 0
        out_dtype = out_dtype or x.dtype
        y = torch.empty((T, layer.hidden), dtype=out_dtype, device=x.device)
        yf = torch.empty((T, layer.hidden), dtype=torch.float32, device=x.device) if want_f32 else None
        if prefill is None:
            prefill = T > 16
        fn = lib().cx_moe_prefill if prefill else lib().cx_moe_decode
        ids = topk_ids.to(torch.int32).contiguous()
        w = topk_w.to(torch.float32).contiguous()
        if isinstance(layer, Q4Layer):
            self._q4_moe(layer, x, ids, w, y, yf)
            return (y, yf) if want_f32 else y
        check(fn(self.handle, layer.handle, x.data_ptr(), cx_dtype(x.dtype), T, ids.data_ptr(),
                 w.data_ptr(), K, y.data_ptr(), cx_dtype(out_dtype), _ptr(yf), self.stream()))
        return (y, yf) if want_f32 else y

    # -- whole-layer wire message (MoeLayerRequest / MoeLayerResponse) -------------
    def moe_layer_request(self, layer: Layer, body: bytes) -> bytes:
        """Runs one MoeLayerRequest body (host bytes, moe_layer_protocol) on
        `layer` and returns the MoeLayerResponse body (host bytes)."""
        if not isinstance(layer, Layer):
            raise TypeError("a whole-layer message runs on a Layer (fp8 experts)")
        info = MoeLayerRequestInfo()
        b = np.frombuffer(body, np.uint8)
        check(lib().cx_moe_layer_request_peek(b.ctypes.data, b.size, C.byref(info)))
        cap = lib().cx_moe_layer_response_size(info.batch_size, info.hidden_dim)
        out = np.empty(cap, np.uint8)
        n = C.c_size_t(0)
        check(lib().cx_moe_layer_request_run(self.handle, layer.handle, b.ctypes.data, b.size,
                                             out.ctypes.data, out.size, C.byref(n)))
        return out[:n.value].tobytes()

    def moe_layer(self, layer: Union[Layer, Q4Layer], x: torch.Tensor, w_router: torch.Tensor, bias: torch.Tensor, *,
                  resident: Optional[torch.Tensor] = None, n_group: int = 8, topk_group: int = 4,
                  top_k: int = 8, norm_topk_prob: bool = True, routed_scaling_factor: float = 2.5,
                  out_dtype: Optional[torch.dtype] = None, want_f32: bool = False, out=None):
        x = x.contiguous()
        T = x.shape[0]
        out_dtype = out_dtype or x.dtype
        if isinstance(layer, Q4Layer):  # its router is a launch of its own, before the layer's
            E, H = layer.n_experts, layer.hidden
            self._q4_ready(layer, x, w_router, bias, resident, *(out or ()))
            w_router, bias = w_router.contiguous(), bias.contiguous()
            resident = None if resident is None else resident.contiguous()
            if w_router.shape != (E, H):
                raise ValueError(f"w_router must be [{E}, {H}], not {list(w_router.shape)}")
            if bias.shape != (E,) or bias.dtype != torch.float32:
                raise ValueError(f"bias must be fp32 [{E}]")
            if resident is not None and (resident.shape != (E,) or resident.element_size() != 1):
                raise ValueError(f"resident must be uint8 [{E}]")
            for t, n, dts in zip(out or (), (H, H, top_k, top_k), (
                    (torch.float16, torch.bfloat16), (torch.float32,), (torch.int32,), (torch.float32,))):
                if t is not None and (t.shape != (T, n) or t.dtype not in dts or not t.is_contiguous()):
                    raise ValueError(f"out must be contiguous: y [{T}, {H}] in 16 bits, its fp32 copy or None, "
                                     f"ids int32 and weights fp32 [{T}, {top_k}]")
        if out is None:
            y = torch.empty((T, layer.hidden), dtype=out_dtype, device=x.device)
            yf = torch.empty((T, layer.hidden), dtype=torch.float32, device=x.device) if want_f32 else None
            ids = torch.empty((T, top_k), dtype=torch.int32, device=x.device)
            w = torch.empty((T, top_k), dtype=torch.float32, device=x.device)
        else:
            y, yf, ids, w = out
        if isinstance(layer, Q4Layer):
            check(lib().cx_route(self.handle, x.data_ptr(), cx_dtype(x.dtype), w_router.data_ptr(),
                                 cx_dtype(w_router.dtype), bias.data_ptr(), _ptr(resident), T, layer.hidden,
                                 layer.n_experts, n_group, topk_group, top_k, int(norm_topk_prob),
                                 routed_scaling_factor, ids.data_ptr(), w.data_ptr(), self.stream()))
            self._q4_moe(layer, x, ids, w, y, yf)
            return y, yf, ids, w
        check(lib().cx_moe_layer(self.handle, layer.handle, x.data_ptr(), cx_dtype(x.dtype), T,
                                 w_router.data_ptr(), cx_dtype(w_router.dtype), bias.data_ptr(),
                                 _ptr(resident), n_group, topk_group, top_k, int(norm_topk_prob),
                                 routed_scaling_factor, y.data_ptr(), cx_dtype(out_dtype), _ptr(yf),
                                 ids.data_ptr(), w.data_ptr(), self.stream()))
        return y, yf, ids, w

    # -- synthetic data ------------------------------------------------------
    def gen_normal(self, seed: int, stream_id: int, shape, std: float, dtype: torch.dtype):
        t = torch.empty(shape, dtype=dtype, device=_device(self.device))
        check(lib().cx_gen_normal(self.handle, seed, stream_id, t.numel(), std, cx_dtype(dtype),
                                  t.data_ptr(), self.stream()))
        return t
