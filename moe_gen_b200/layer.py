"""Host-side MoE layer object: owns the native handle, the packed weight buffer and
the workspace (all torch CUDA tensors — torch is used for device memory and streams
only), and calls the C ABI for every computation.

The staged methods mirror the steps of the reference's layer
(moe_gen/models/deepseek/deepseekv3/modeling_deepseek_v3.py: MoEGate.forward
:500-561, DeepseekV3MoE.moe_infer :628-711) so tests can compare stage by stage.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools
from typing import Optional, Tuple

import torch

from . import lib as L


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _whole(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and on a 16-byte boundary, as the kernels read rows: a copy where it is a view that begins elsewhere."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# Sizes are asked for once: a call of the library costs a microsecond, a tenth of an adapter call.
@functools.lru_cache(maxsize=1024)
def _plan_bytes(rows: int, n_adapters: int) -> int:
    size = C.c_size_t()
    L.check(L.load().mg_adapter_plan_bytes(rows, n_adapters, C.byref(size)))
    return size.value


@functools.lru_cache(maxsize=None)
def _rank_stride(rank: int) -> int:
    n = C.c_int32()
    L.check(L.load().mg_adapter_rank_stride(rank, C.byref(n)))
    return n.value


class AdapterPlan:
    """Rows sorted by their adapters (MoELayer.adapter_plan, .adapter_plan_sorted), for every adapter call on these rows."""
    __slots__ = ("buf", "rows", "n_adapters")

    def __init__(self, buf: torch.Tensor, rows: int, n_adapters: int):
        self.buf, self.rows, self.n_adapters = buf, rows, n_adapters


_NO_SWITCH = contextlib.nullcontext()
_raw_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


class MoELayer:
    def __init__(self, *, hidden: int, inter: int, n_experts: int, top_k: int, inter_shared: int = 0,
                 n_group: int = 1, topk_group: int = 1, gating: int = L.GATE_SOFTMAX_GREEDY,
                 norm_topk_prob: bool = False, routed_scale: float = 1.0,
                 weight_format: int = L.WEIGHT_BF16, combine_mode: int = L.COMBINE_FP32,
                 ep_rank: int = 0, ep_size: int = 1, device=None):
        if not torch.cuda.is_available():
            raise RuntimeError("moe_gen_b200 needs a CUDA device (sm_100a); there is no CPU path")
        self.lib = L.load()
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self._index = torch.cuda.current_device() if self.device.index is None else self.device.index
        self.desc = L.LayerDesc(C.sizeof(L.LayerDesc), hidden, inter, inter_shared, n_experts, top_k, n_group,
                                topk_group, gating, int(bool(norm_topk_prob)), float(routed_scale),
                                weight_format, combine_mode, ep_rank, ep_size)
        self.H, self.I, self.Is, self.E, self.k = hidden, inter, inter_shared, n_experts, top_k
        self.e_local = n_experts // ep_size
        self.expert_lo = ep_rank * self.e_local
        self._h = C.c_void_p()
        with self._on_device():
            L.check(self.lib.mg_create(C.byref(self.desc), C.byref(self._h)))
            n = C.c_size_t()
            L.check(self.lib.mg_packed_weight_bytes(self._h, C.byref(n)))
            # zeroed: the alignment gaps between its sections are never written
            self.packed = torch.zeros(n.value, dtype=torch.uint8, device=self.device)
        self.gate_w: Optional[torch.Tensor] = None
        self.bias: Optional[torch.Tensor] = None
        self._ws: Optional[torch.Tensor] = None
        self._ws_tokens = -1
        self._captured: list = []               # buffers that captured graphs go on using
        self.options = {}                       # option id -> last value set

    # ------------------------------------------------------------------ lifetime
    def close(self):
        if getattr(self, "_h", None) is not None and self._h.value:
            self.lib.mg_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # Entering torch.cuda.device and asking for torch.cuda.current_stream() takes 1.5 and 3.3 us of a call whose launch takes 3:
    # the device is set where it is another one only, and the stream's handle is read without making a Stream of it.
    def _on_device(self):
        return _NO_SWITCH if _raw_device() == self._index else torch.cuda.device(self._index)

    def _stream(self) -> int:
        return _raw_stream(self._index)

    def _check_in(self, t: torch.Tensor, dtype, what: str):
        if t.device != self.device or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{what}: expected contiguous {dtype} tensor on {self.device}, got "
                             f"{t.dtype} on {t.device} contiguous={t.is_contiguous()}")

    def _check_out(self, out: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
        self._check_in(out, like.dtype, "out")
        if out.numel() != like.numel():
            raise ValueError(f"out: {tuple(out.shape)} for results of {tuple(like.shape)}")
        return out

    # ------------------------------------------------------------------ weights
    def set_router(self, gate_weight: torch.Tensor, bias: Optional[torch.Tensor] = None):
        """gate.weight [E,H] (kept as bf16) and, for noaux_tc, e_score_correction_bias [E] (fp32)."""
        self.gate_w = _whole(gate_weight.detach().to(self.device, torch.bfloat16))
        assert self.gate_w.shape == (self.E, self.H)
        self.bias = None if bias is None else bias.detach().to(self.device, torch.float32).contiguous()

    def load_expert(self, local_expert: int, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                    scales: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None):
        """Packs one expert ([I,H], [I,H], [H,I] as nn.Linear stores them).  local_expert = -1 is
        the shared expert.  FP8 layers pass float8_e4m3fn matrices plus their fp32 scales; int8 layers, for the shared
        expert too, int8 matrices plus the fp32 scales of their rows ([I], [I], [H])."""
        fp8 = self.desc.weight_format == L.WEIGHT_FP8_BLOCK128 and local_expert >= 0
        int8 = self.desc.weight_format == L.WEIGHT_INT8_CHANNEL
        dt = torch.float8_e4m3fn if fp8 else torch.int8 if int8 else torch.bfloat16
        mats = [_whole(m.detach().to(self.device)) for m in (gate, up, down)]
        I = self.Is if local_expert < 0 else self.I
        for m, shp in zip(mats, ((I, self.H), (I, self.H), (self.H, I))):
            if m.dtype != dt or tuple(m.shape) != shp:
                raise ValueError(f"expert matrix {tuple(m.shape)} {m.dtype}, expected {shp} {dt}")
        sc = [None, None, None]
        if fp8:
            if scales is None:
                raise ValueError("FP8 layer: scales=(gate_scale, up_scale, down_scale) required")
            sc = [s.detach().to(self.device, torch.float32).contiguous() for s in scales]
        if int8:
            if scales is None or any(s is None for s in scales):
                raise ValueError("int8 layer: scales=(gate_scale, up_scale, down_scale) required")
            sc = [s.detach().to(self.device, torch.float32).reshape(-1).contiguous() for s in scales]
            for s, m in zip(sc, mats):
                if s.numel() != m.shape[0]:
                    raise ValueError(f"int8 expert matrix of {m.shape[0]} rows with {s.numel()} scales")
        with self._on_device():
            L.check(self.lib.mg_pack_expert(self._h, local_expert, mats[0].data_ptr(), mats[1].data_ptr(),
                                            mats[2].data_ptr(), _ptr(sc[0]), _ptr(sc[1]), _ptr(sc[2]),
                                            self.packed.data_ptr(), self._stream()))
            torch.cuda.current_stream().synchronize()   # sources may be temporaries

    def load_shared(self, gate, up, down, scales: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None):
        self.load_expert(-1, gate, up, down, scales)

    # ------------------------------------------------------------------ sizes
    def padded_rows(self, n_rows: int) -> int:
        out = C.c_int64()
        L.check(self.lib.mg_padded_rows(self._h, n_rows, C.byref(out)))
        return out.value

    def _kept(self, buf: torch.Tensor) -> torch.Tensor:
        """buf, kept for the layer's life where the call is being captured: a graph writes to it at every replay, also after a larger
        batch has been given another."""
        with self._on_device():
            if torch.cuda.is_current_stream_capturing() and all(b is not buf for b in self._captured):
                self._captured.append(buf)
        return buf

    def _workspace(self, T: int) -> torch.Tensor:
        if self._ws is None or T > self._ws_tokens:
            n = C.c_size_t()
            L.check(self.lib.mg_workspace_bytes(self._h, T, 0, C.byref(n)))
            self._ws = None
            self._ws = torch.empty(max(n.value, 256), dtype=torch.uint8, device=self.device)
            self._ws_tokens = T
        return self._kept(self._ws)

    def workspace_view(self, which: int, T: int) -> int:
        p = C.c_void_p()
        L.check(self.lib.mg_workspace_ptr(self._h, self._ws.data_ptr(), self._ws_tokens, 0, which, C.byref(p)))
        return p.value

    def device_status(self) -> Tuple[int, int]:
        code, detail = C.c_int32(), C.c_int32()
        L.check(self.lib.mg_device_status(self._h, C.byref(code), C.byref(detail)))
        return code.value, detail.value

    def set_option(self, option: int, value: int):
        L.check(self.lib.mg_set_option(self._h, option, value))
        self.options[option] = value
        if option != L.OPT_KEEP_DEQUANT:
            self._ws, self._ws_tokens = None, -1    # workspace layout may depend on options
            self._hws = None

    def set_stage_timing(self, enable: bool):
        """Record the stages' times; forwards then follow another schedule (mg_set_stage_timing), with the same bits."""
        L.check(self.lib.mg_set_stage_timing(self._h, int(enable)))

    def stage_times(self) -> dict:
        """Milliseconds per stage of the last forward (call after synchronising)."""
        ms = (C.c_float * len(L.STAGES))()
        L.check(self.lib.mg_stage_times(self._h, ms, len(L.STAGES)))
        return dict(zip(L.STAGES, [float(v) for v in ms]))

    def last_launch_count(self) -> int:
        n = C.c_int32()
        L.check(self.lib.mg_last_launch_count(self._h, C.byref(n)))
        return n.value

    # ------------------------------------------------------------------ whole layer
    def forward(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x: [..., H] bf16 on the layer's device -> same shape.  Asynchronous on the current stream.  A layer's forwards share its
        workspace: they follow one another on the GPU, replays of captured ones included."""
        shape = x.shape
        x2 = x.reshape(-1, self.H)
        self._check_in(x2, torch.bfloat16, "hidden_states")
        T = x2.shape[0]
        ws = self._workspace(T)
        y = torch.empty_like(x2) if out is None else self._check_out(out, x2)
        with self._on_device():
            L.check(self.lib.mg_moe_forward(self._h, x2.data_ptr(), T, self.gate_w.data_ptr(), _ptr(self.bias),
                                            self.packed.data_ptr(), ws.data_ptr(), ws.numel(), y.data_ptr(),
                                            self._stream()))
        return y.view(shape)

    __call__ = forward

    def forward_from_logits(self, x: torch.Tensor, logits: torch.Tensor, out: Optional[torch.Tensor] = None):
        """The layer on router logits the caller computed ([T,E] fp32, e.g. F.linear(x.float(),
        W.float()) as the reference's MoEGate does, modeling_deepseek_v3.py:503-508): the routing is
        then an exact function of those logits."""
        shape = x.shape
        x2 = x.reshape(-1, self.H)
        self._check_in(x2, torch.bfloat16, "hidden_states")
        self._check_in(logits, torch.float32, "logits")
        T = x2.shape[0]
        if tuple(logits.shape) != (T, self.E):
            raise ValueError(f"logits {tuple(logits.shape)}, expected {(T, self.E)}")
        ws = self._workspace(T)
        y = torch.empty_like(x2) if out is None else self._check_out(out, x2)
        with self._on_device():
            L.check(self.lib.mg_moe_forward_from_logits(self._h, x2.data_ptr(), T, logits.data_ptr(), _ptr(self.bias),
                                                        self.packed.data_ptr(), ws.data_ptr(), ws.numel(),
                                                        y.data_ptr(), self._stream()))
        return y.view(shape)

    # ------------------------------------------------------------------ decoder-layer glue
    def rmsnorm(self, x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """weight * bf16(x * rsqrt(mean(x^2) + eps)): the reference's DeepseekV3RMSNorm
        (modeling_deepseek_v3.py:125-150) with the bf16 weight of a bfloat16 model."""
        x2 = x.reshape(-1, self.H)
        self._check_in(x2, torch.bfloat16, "hidden_states")
        self._check_in(weight, torch.bfloat16, "norm weight")
        if weight.numel() != self.H:
            raise ValueError(f"norm weight has {weight.numel()} elements, hidden size is {self.H}")
        y = torch.empty_like(x2) if out is None else self._check_out(out, x2)
        with self._on_device():
            L.check(self.lib.mg_rmsnorm(self._h, x2.data_ptr(), weight.data_ptr(), float(eps), x2.shape[0],
                                        y.data_ptr(), self._stream()))
        return y.view(x.shape)

    def _norm_args(self, x, residual, weight, sum_out):
        """Rows, columns and strides of x, the residual and their sum; the sum's tensor."""
        n, cols, ldx = self._rows_of(x, torch.bfloat16, "x")
        self._check_in(weight, torch.bfloat16, "norm weight")
        if weight.numel() != cols:
            raise ValueError(f"norm weight has {weight.numel()} elements, rows have {cols}")
        if residual is None:
            if sum_out is not None:
                raise ValueError("sum_out: there is no residual to add")
            return n, cols, ldx, 0, x, 0
        nr, rcols, ldr = self._rows_of(residual, torch.bfloat16, "residual")
        if (nr, rcols) != (n, cols):
            raise ValueError(f"residual {tuple(residual.shape)} for rows of {tuple(x.shape)}")
        sum_out, lds = self._out_rows(sum_out, n, cols, "sum_out", x, ldx)
        return n, cols, ldx, ldr, sum_out, lds

    def _out_rows(self, out: Optional[torch.Tensor], n: int, cols: int, what: str, like: torch.Tensor, ld_like: int):
        """out and the elements between its rows; a new one has its rows on 16-byte boundaries (as those of `like`, bf16 rows of
        n and cols ld_like apart, where these do: the cheaper allocation)."""
        if out is None:
            if ld_like == cols and cols % 8 == 0:
                return torch.empty_like(like), cols
            ld = (cols + 7) // 8 * 8
            return torch.empty_strided((n, cols), (ld, 1), dtype=torch.bfloat16, device=self.device), ld
        rows, o_cols, ld = self._rows_of(out, torch.bfloat16, what)
        if (rows, o_cols) != (n, cols):
            raise ValueError(f"{what} {tuple(out.shape)}, expected {(n, cols)}")
        return out, ld

    def add_rmsnorm(self, x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                    out: Optional[torch.Tensor] = None, sum_out: Optional[torch.Tensor] = None):
        """-> (y, h) with h = bf16(x + residual), y = bf16(weight * h * rsqrt(mean(h^2) + eps)), in one launch; h = x without a residual.
        y is rounded once, where rmsnorm rounds a second time before the weight.  x, residual and weight bf16, [rows, cols] with
        adjacent columns (any cols, rows may lie further apart).  out and sum_out may each be x or the residual,
        not one another, and overlap nothing otherwise.  Any layer serves."""
        n, cols, ldx, ldr, h, lds = self._norm_args(x, residual, weight, sum_out)
        y, ldo = self._out_rows(out, n, cols, "out", x, ldx)
        with self._on_device():
            L.check(self.lib.mg_add_rmsnorm(self._h, x.data_ptr(), ldx, _ptr(residual), ldr, weight.data_ptr(), eps, n, cols,
                                            None if residual is None else h.data_ptr(), lds, y.data_ptr(), ldo, self._stream()))
        return y, h

    def add_rmsnorm_int8(self, x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                         sum_out: Optional[torch.Tensor] = None):
        """-> (q, scale, h): add_rmsnorm with its rows quantised as quantize_rows does (int8 on 128-byte strides, fp32 scales), from
        their fp32 values; what int8_matmul and permute_rows_int8 take."""
        n, cols, ldx, ldr, h, lds = self._norm_args(x, residual, weight, sum_out)
        ldq = (cols + 127) // 128 * 128
        q = torch.empty_strided((n, cols), (ldq, 1), dtype=torch.int8, device=self.device)
        scale = torch.empty(n, dtype=torch.float32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_add_rmsnorm_int8(self._h, x.data_ptr(), ldx, _ptr(residual), ldr, weight.data_ptr(), eps, n, cols,
                                                 None if residual is None else h.data_ptr(), lds, q.data_ptr(), ldq, scale.data_ptr(),
                                                 self._stream()))
        return q, scale, h

    def add_rmsnorm_grad(self, grad_y: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                         grad_h: Optional[torch.Tensor] = None, need_x: bool = True, need_w: bool = True):
        """Gradients of add_rmsnorm for grad_y and for grad_h, which reaches h by other ways -> (grad_x, which is the residual's too,
        bf16; grad_weight [cols] fp32), None for the one that is not needed.  At most 16384 columns."""
        n, cols, ldh = self._rows_of(h, torch.bfloat16, "h")
        self._check_in(weight, torch.bfloat16, "norm weight")
        if weight.numel() != cols:
            raise ValueError(f"norm weight has {weight.numel()} elements, rows have {cols}")
        ng, gcols, ldgy = self._rows_of(grad_y, torch.bfloat16, "grad_y")
        nh, hcols, ldgh = (n, cols, 0) if grad_h is None else self._rows_of(grad_h, torch.bfloat16, "grad_h")
        if (ng, gcols) != (n, cols) or (nh, hcols) != (n, cols):
            raise ValueError(f"gradients of {(ng, gcols)} and {(nh, hcols)} for rows of {(n, cols)}")
        gx, ldgx = self._out_rows(None, n, cols, "grad_x", h, ldh) if need_x else (None, 0)
        if not (need_x or need_w):
            return None, None
        gw = torch.empty(cols, dtype=torch.float32, device=self.device) if need_w else None
        ws, size = None, 0
        if need_w and n > L.NORM_GRAD_FEW:
            need = C.c_size_t()
            L.check(self.lib.mg_add_rmsnorm_grad_ws_bytes(self._h, n, cols, C.byref(need)))
            size = need.value
            ws = torch.empty(size, dtype=torch.uint8, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_add_rmsnorm_grad(self._h, grad_y.data_ptr(), ldgy, h.data_ptr(), ldh, weight.data_ptr(), eps, n, cols,
                                                 _ptr(grad_h), ldgh, _ptr(gx), ldgx, _ptr(gw), _ptr(ws), size, self._stream()))
        return gx, gw

    def block_forward(self, hidden: torch.Tensor, norm_weight: torch.Tensor, eps: float = 1e-6,
                      out: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """hidden + moe(rmsnorm(hidden)): the decoder layer's second half
        (modeling_deepseek_v3.py:1361-1365) with the residual add done by the combine kernel.
        out may be hidden itself (in-place update of the residual stream).  With a residual (same shape) the block runs on
        bf16(hidden + residual), as if that had been handed in, added by the norm's launch; out may be either."""
        shape = hidden.shape
        h2 = hidden.reshape(-1, self.H)
        self._check_in(h2, torch.bfloat16, "hidden_states")
        self._check_in(norm_weight, torch.bfloat16, "norm weight")
        if norm_weight.numel() != self.H:
            raise ValueError(f"norm weight has {norm_weight.numel()} elements, hidden size is {self.H}")
        T = h2.shape[0]
        ws = self._workspace(T)
        if getattr(self, "_xnorm", None) is None or self._xnorm.shape[0] < T:
            self._xnorm = torch.empty(max(T, 1), self.H, dtype=torch.bfloat16, device=self.device)
        xnorm = self._kept(self._xnorm)
        y = torch.empty_like(h2) if out is None else self._check_out(out, h2)
        if residual is not None:
            self._check_in(residual, torch.bfloat16, "residual")
            if residual.shape != shape:
                raise ValueError(f"residual {tuple(residual.shape)} for hidden states of {tuple(shape)}")
            with self._on_device():
                L.check(self.lib.mg_moe_block_forward_add(self._h, h2.data_ptr(), residual.data_ptr(), norm_weight.data_ptr(), float(eps), T,
                                                          self.gate_w.data_ptr(), _ptr(self.bias), self.packed.data_ptr(),
                                                          xnorm.data_ptr(), ws.data_ptr(), ws.numel(), y.data_ptr(), self._stream()))
            return y.view(shape)
        with self._on_device():
            L.check(self.lib.mg_moe_block_forward(self._h, h2.data_ptr(), norm_weight.data_ptr(), float(eps), T,
                                                  self.gate_w.data_ptr(), _ptr(self.bias), self.packed.data_ptr(),
                                                  xnorm.data_ptr(), ws.data_ptr(), ws.numel(), y.data_ptr(),
                                                  self._stream()))
        return y.view(shape)

    @staticmethod
    def host_chunks(T: int, chunk_tokens: int) -> list:
        """Token counts of the chunks the host-buffer forward uses (mg_host_chunk_plan): the copy-in of
        the first chunk and the copy-out of the last one cannot overlap with compute, so those two are
        half a chunk; the ones between them are one and a half, because every chunk streams all expert
        weights once."""
        lib = L.load()
        n = C.c_int32()
        L.check(lib.mg_host_chunk_plan(T, max(1, chunk_tokens), None, 0, C.byref(n)))
        sizes = (C.c_int64 * max(n.value, 1))()
        L.check(lib.mg_host_chunk_plan(T, max(1, chunk_tokens), sizes, n.value, C.byref(n)))
        return [int(v) for v in sizes[:n.value]]

    def forward_host(self, x_host: torch.Tensor, y_host: Optional[torch.Tensor] = None,
                     chunk_tokens: int = 8192) -> torch.Tensor:
        """Host-buffer entry (mg_moe_forward_host): x_host [T,H] bf16 in (preferably pinned) host memory
        -> y_host.  The library copies chunks in, computes and copies out on three streams; returns
        after the last copy has finished."""
        T = x_host.shape[0]
        if x_host.dtype != torch.bfloat16 or not x_host.is_contiguous() or x_host.is_cuda:
            raise ValueError("x_host: expected a contiguous bfloat16 tensor in host memory")
        if y_host is None:
            y_host = torch.empty_like(x_host, pin_memory=x_host.is_pinned())
        if T == 0:
            return y_host
        with self._on_device():
            n = C.c_size_t()
            L.check(self.lib.mg_host_workspace_bytes(self._h, T, chunk_tokens, C.byref(n)))
            if getattr(self, "_hws", None) is None or self._hws.numel() < n.value:
                self._hws = None
                self._hws = torch.empty(n.value, dtype=torch.uint8, device=self.device)
            L.check(self.lib.mg_moe_forward_host(self._h, x_host.data_ptr(), T, self.gate_w.data_ptr(), _ptr(self.bias),
                                                 self.packed.data_ptr(), self._hws.data_ptr(), self._hws.numel(),
                                                 y_host.data_ptr(), chunk_tokens, self._stream()))
            torch.cuda.current_stream().synchronize()
        return y_host

    # ------------------------------------------------------------------ stages
    def gate_logits(self, x: torch.Tensor) -> torch.Tensor:
        self._check_rows(x, torch.bfloat16, None, self.H, "hidden_states")
        T = x.shape[0]
        logits = torch.empty(T, self.E, dtype=torch.float32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_gate_logits(self._h, x.data_ptr(), self.gate_w.data_ptr(), T, logits.data_ptr(),
                                            self._stream()))
        return logits

    def route_topk(self, logits: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        self._check_rows(logits, torch.float32, None, self.E, "logits")
        T = logits.shape[0]
        idx = torch.empty(T, self.k, dtype=torch.int32, device=self.device)
        w = torch.empty(T, self.k, dtype=torch.float32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_route_topk(self._h, logits.data_ptr(), _ptr(self.bias), T, idx.data_ptr(),
                                           w.data_ptr(), self._stream()))
        return idx, w

    def gate_route(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """The routing mg_moe_forward uses: router product on the tensor cores, top-k, and near-tie tokens
        re-routed from exactly recomputed logits.  -> topk_idx, topk_w, logits (recomputed entries included),
        fix (int32: [0] tokens routed again, [1] of which with the whole row recomputed, [2] single logits
        recomputed; tokens from [4], row tokens from [4+T], (token, expert) pairs from [4+2T])."""
        self._check_rows(x, torch.bfloat16, None, self.H, "hidden_states")
        T = x.shape[0]
        logits = torch.empty(T, self.E, dtype=torch.float32, device=self.device)
        idx = torch.empty(T, self.k, dtype=torch.int32, device=self.device)
        w = torch.empty(T, self.k, dtype=torch.float32, device=self.device)
        n = C.c_size_t()
        L.check(self.lib.mg_route_fix_bytes(T, C.byref(n)))
        fix = torch.zeros(n.value // 4, dtype=torch.int32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_gate_route_topk(self._h, x.data_ptr(), self.gate_w.data_ptr(), _ptr(self.bias), T,
                                                logits.data_ptr(), idx.data_ptr(), w.data_ptr(), fix.data_ptr(),
                                                self._stream()))
        return idx, w, logits, fix

    def permute_plan(self, topk_idx: torch.Tensor, expert_lo: int = 0, n_plan: Optional[int] = None):
        """-> counts [n], offsets [n+1], pad_offsets [n+1], dst_row [T,k] (all int32)."""
        self._check_rows(topk_idx, torch.int32, None, self.k, "topk_idx")
        n = self.E if n_plan is None else n_plan
        T = topk_idx.shape[0]
        dev = self.device
        counts = torch.empty(n, dtype=torch.int32, device=dev)
        offsets = torch.empty(n + 1, dtype=torch.int32, device=dev)
        pad = torch.empty(n + 1, dtype=torch.int32, device=dev)
        dst = torch.empty(T, self.k, dtype=torch.int32, device=dev)
        nb = C.c_size_t()
        L.check(self.lib.mg_plan_ws_bytes(self._h, T, C.byref(nb)))
        ws = torch.empty(max(nb.value, 4), dtype=torch.uint8, device=dev)
        with self._on_device():
            L.check(self.lib.mg_permute_plan(self._h, topk_idx.data_ptr(), T, expert_lo, n, counts.data_ptr(),
                                             offsets.data_ptr(), pad.data_ptr(), dst.data_ptr(), ws.data_ptr(),
                                             self._stream()))
        return counts, offsets, pad, dst

    def _check_plan(self, dst_row: torch.Tensor, counts: torch.Tensor, pad_offsets: torch.Tensor):
        self._check_in(counts, torch.int32, "counts")
        self._check_in(pad_offsets, torch.int32, "pad_offsets")
        if counts.numel() > self.E or pad_offsets.numel() != counts.numel() + 1:
            raise ValueError(f"counts of {counts.numel()} and pad_offsets of {pad_offsets.numel()} entries for {self.E} experts")

    def _check_rows(self, t: torch.Tensor, dtype, rows: Optional[int], cols: int, what: str):
        self._check_in(t, dtype, what)
        shape = t.shape
        if len(shape) != 2 or shape[1] != cols or (rows is not None and shape[0] != rows):
            raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {('rows' if rows is None else rows, cols)}")

    def permute_rows(self, x: torch.Tensor, dst_row: torch.Tensor, rows_padded: int, counts: Optional[torch.Tensor] = None,
                     pad_offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
        """perm[dst_row[t, j]] = x[t], zeros in the rows no pick points at.  With the plan's counts and pad_offsets only those
        rows are written as zeros, in the same launch, instead of all rows before it (a plan of distinct experts per token: one
        that a token names twice leaves a counted row without a pick, which then stays as it was)."""
        if counts is not None and pad_offsets is not None:
            self._check_rows(x, torch.bfloat16, None, self.H, "hidden_states")
            self._check_rows(dst_row, torch.int32, x.shape[0], self.k, "dst_row")
            self._check_plan(dst_row, counts, pad_offsets)
            perm = torch.empty(rows_padded, self.H, dtype=torch.bfloat16, device=self.device)
            with self._on_device():
                L.check(self.lib.mg_permute_rows_padded(self._h, x.data_ptr(), dst_row.data_ptr(), x.shape[0],
                                                        counts.data_ptr(), pad_offsets.data_ptr(), counts.numel(), rows_padded,
                                                        perm.data_ptr(), self._stream()))
            return perm
        self._check_rows(x, torch.bfloat16, None, self.H, "hidden_states")
        self._check_rows(dst_row, torch.int32, x.shape[0], self.k, "dst_row")
        perm = torch.zeros(rows_padded, self.H, dtype=torch.bfloat16, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_permute_rows_bounded(self._h, x.data_ptr(), None, dst_row.data_ptr(), x.shape[0], rows_padded,
                                                     perm.data_ptr(), None, self._stream()))
        return perm

    def permute_rows_grad(self, grad_rows: torch.Tensor, dst_row: torch.Tensor) -> torch.Tensor:
        """Gradient of permute_rows: grad_x[t] = sum_j grad_rows[dst_row[t, j]] (fp32 sum, one rounding).  Entries of dst_row that
        are negative or not below grad_rows' rows are left out."""
        self._check_rows(grad_rows, torch.bfloat16, None, self.H, "grad_rows")
        self._check_rows(dst_row, torch.int32, None, self.k, "dst_row")
        T = dst_row.shape[0]
        gx = torch.empty(T, self.H, dtype=torch.bfloat16, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_permute_rows_grad_bounded(self._h, grad_rows.data_ptr(), grad_rows.shape[0], dst_row.data_ptr(), T,
                                                          gx.data_ptr(), self._stream()))
        return gx

    def combine_grad(self, grad_y: torch.Tensor, out_rows: torch.Tensor, dst_row: torch.Tensor, topk_w: torch.Tensor,
                     counts: torch.Tensor, pad_offsets: torch.Tensor, need_rows: bool = True, need_w: bool = True):
        """Gradients of combine's sum -> (grad_rows like out_rows, zeros where no pick points, by a plan of distinct experts per
        token as in permute_rows; grad_w [T, k] fp32), None for the one that is not needed.  The gradient of shared_out is
        grad_y itself."""
        T = dst_row.shape[0]
        self._check_rows(grad_y, torch.bfloat16, T, self.H, "grad_y")
        self._check_rows(out_rows, torch.bfloat16, None, self.H, "out_rows")
        self._check_rows(dst_row, torch.int32, T, self.k, "dst_row")
        self._check_rows(topk_w, torch.float32, T, self.k, "topk_w")
        self._check_plan(dst_row, counts, pad_offsets)
        grows = torch.empty_like(out_rows) if need_rows else None
        gw = torch.empty(T, self.k, dtype=torch.float32, device=self.device) if need_w else None
        with self._on_device():
            L.check(self.lib.mg_combine_grad(self._h, grad_y.data_ptr(), out_rows.data_ptr(), dst_row.data_ptr(), topk_w.data_ptr(),
                                             T, counts.data_ptr(), pad_offsets.data_ptr(), counts.numel(), out_rows.shape[0],
                                             _ptr(grows), _ptr(gw), self._stream()))
        return grows, gw

    def route_topk_grad(self, logits: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor,
                        grad_w: torch.Tensor) -> torch.Tensor:
        """Gradient of route_topk's weights with respect to the logits, the picks being constants: [T, E] fp32."""
        T = logits.shape[0]
        self._check_rows(logits, torch.float32, None, self.E, "logits")
        self._check_rows(topk_idx, torch.int32, T, self.k, "topk_idx")
        self._check_rows(topk_w, torch.float32, T, self.k, "topk_w")
        self._check_rows(grad_w, torch.float32, T, self.k, "grad_w")
        gl = torch.empty(T, self.E, dtype=torch.float32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_route_topk_grad(self._h, logits.data_ptr(), topk_idx.data_ptr(), topk_w.data_ptr(),
                                                grad_w.data_ptr(), T, gl.data_ptr(), self._stream()))
        return gl

    # ------------------------------------------------------------------ 8-bit integers
    def _rows_of(self, t: torch.Tensor, dtype, what: str) -> Tuple[int, int, int]:
        """Rows, columns and elements between rows of a [rows, cols] tensor whose columns are adjacent; rows may lie further apart.
        torch leaves the stride of a single row open: enough is named for it to pass for one on any boundary."""
        if t.dtype != dtype or t.dim() != 2 or t.device != self.device:
            raise ValueError(f"{what}: expected a [rows, cols] {dtype} tensor on {self.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
        n, cols = t.shape
        step, inner = t.stride()
        if cols > 1 and inner != 1:
            raise ValueError(f"{what}: the elements of a row must be adjacent (strides {t.stride()})")
        return n, cols, step if n > 1 else (cols + 15) // 16 * 16

    def quantize_rows(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Rows of bf16 -> (q [rows, cols] int8 with rows on 128-byte strides, scale [rows] fp32): the values are q * scale.
        A row that holds an infinity or a NaN has scale NaN and q 0."""
        n, cols, ldx = self._rows_of(x, torch.bfloat16, "x")
        ldq = (cols + 127) // 128 * 128
        q = torch.empty_strided((n, cols), (ldq, 1), dtype=torch.int8, device=self.device)
        scale = torch.empty(n, dtype=torch.float32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_quantize_rows_int8(self._h, x.data_ptr(), n, cols, ldx, q.data_ptr(), ldq, scale.data_ptr(),
                                                   self._stream()))
        return q, scale

    def _int8_args(self, wq: torch.Tensor, w_scale: torch.Tensor, cols: int, n_rows: int, out: Optional[torch.Tensor]):
        n_out, w_cols, ldw = self._rows_of(wq, torch.int8, "wq")
        if w_cols != cols:
            raise ValueError(f"wq {tuple(wq.shape)} for rows of {cols}")
        self._check_in(w_scale, torch.float32, "w_scale")
        if w_scale.numel() != n_out:
            raise ValueError(f"{w_scale.numel()} scales for {n_out} output channels")
        if out is None:
            ldo = (n_out + 7) // 8 * 8
            return n_out, ldw, torch.empty_strided((n_rows, n_out), (ldo, 1), dtype=torch.bfloat16, device=self.device), ldo
        rows, o_cols, ldo = self._rows_of(out, torch.bfloat16, "out")
        if (rows, o_cols) != (n_rows, n_out):
            raise ValueError(f"out {tuple(out.shape)}, expected {(n_rows, n_out)}")
        return n_out, ldw, out, ldo

    def int8_matmul(self, xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """bf16(float(xq . wq^T) * x_scale[row] * w_scale[column]): xq [rows, cols] and wq [n_out, cols] int8 with rows on 16-byte
        boundaries (views of wider tensors will do; quantize_rows gives such rows), fp32 scales.  Any layer serves."""
        n, cols, ldx = self._rows_of(xq, torch.int8, "xq")
        self._check_in(x_scale, torch.float32, "x_scale")
        if x_scale.numel() != n:
            raise ValueError(f"{x_scale.numel()} scales for {n} rows")
        n_out, ldw, out, ldo = self._int8_args(wq, w_scale, cols, n, out)
        with self._on_device():
            L.check(self.lib.mg_int8_matmul(self._h, xq.data_ptr(), ldx, x_scale.data_ptr(), n, wq.data_ptr(), ldw,
                                            w_scale.data_ptr(), n_out, cols, out.data_ptr(), ldo, self._stream()))
        return out

    def int8_linear(self, x: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """int8_matmul of bf16 rows x, quantised per token (quantize_rows) in the same call."""
        n, cols, ldx = self._rows_of(x, torch.bfloat16, "x")
        n_out, ldw, out, ldo = self._int8_args(wq, w_scale, cols, n, out)
        need = C.c_size_t()
        L.check(self.lib.mg_int8_linear_ws_bytes(n, n_out, cols, C.byref(need)))
        size = need.value
        ws = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        with self._on_device():
            L.check(self.lib.mg_int8_linear(self._h, x.data_ptr(), ldx, n, wq.data_ptr(), ldw, w_scale.data_ptr(), n_out, cols,
                                            _ptr(ws), size, out.data_ptr(), ldo, self._stream()))
        return out

    def permute_rows_int8(self, xq: torch.Tensor, x_scale: torch.Tensor, dst_row: torch.Tensor, rows_padded: int):
        """-> expert-sorted quantised rows [rows_padded, H] and their scales; rows no pick points at are left open."""
        self._check_rows(xq, torch.int8, None, self.H, "xq")
        self._check_in(x_scale, torch.float32, "x_scale")
        self._check_rows(dst_row, torch.int32, xq.shape[0], self.k, "dst_row")
        if x_scale.numel() != xq.shape[0]:
            raise ValueError(f"{x_scale.numel()} scales for {xq.shape[0]} rows")
        q = torch.empty(rows_padded, self.H, dtype=torch.int8, device=self.device)
        s = torch.empty(rows_padded, dtype=torch.float32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_permute_rows_bounded(self._h, xq.data_ptr(), x_scale.data_ptr(), dst_row.data_ptr(), xq.shape[0],
                                                     rows_padded, q.data_ptr(), s.data_ptr(), self._stream()))
        return q, s

    def expert_ffn_int8(self, perm_q: torch.Tensor, perm_scale: torch.Tensor, pad_offsets: torch.Tensor, counts: torch.Tensor,
                        dst_row: torch.Tensor):
        """-> (h_buf [rows, I] bf16, out_rows [rows, H] bf16) of an int8 layer's experts; zeros in the rows no pick points at."""
        rows = perm_q.shape[0]
        self._check_rows(perm_q, torch.int8, None, self.H, "perm_q")
        self._check_in(perm_scale, torch.float32, "perm_scale")
        self._check_rows(dst_row, torch.int32, None, self.k, "dst_row")
        self._check_plan(dst_row, counts, pad_offsets)
        if perm_scale.numel() != rows or counts.numel() != self.e_local:
            raise ValueError(f"{perm_scale.numel()} scales for {rows} rows, {counts.numel()} counts for {self.e_local} experts")
        hbuf = torch.zeros(rows, self.I, dtype=torch.bfloat16, device=self.device)
        out = torch.zeros(rows, self.H, dtype=torch.bfloat16, device=self.device)
        hq = torch.empty(rows, self.I, dtype=torch.int8, device=self.device)
        hs = torch.empty(rows, dtype=torch.float32, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_expert_ffn_int8(self._h, perm_q.data_ptr(), perm_scale.data_ptr(), pad_offsets.data_ptr(),
                                                counts.data_ptr(), rows, dst_row.data_ptr(), dst_row.shape[0],
                                                self.packed.data_ptr(), hbuf.data_ptr(), hq.data_ptr(), hs.data_ptr(),
                                                out.data_ptr(), self._stream()))
        return hbuf, out

    def shared_ffn_int8(self, xq: torch.Tensor, x_scale: torch.Tensor) -> torch.Tensor:
        self._check_rows(xq, torch.int8, None, self.H, "xq")
        self._check_in(x_scale, torch.float32, "x_scale")
        T = xq.shape[0]
        if x_scale.numel() != T:
            raise ValueError(f"{x_scale.numel()} scales for {T} rows")
        hs = torch.empty(T, self.Is, dtype=torch.bfloat16, device=self.device)
        hq = torch.empty(T, self.Is, dtype=torch.int8, device=self.device)
        sc = torch.empty(T, dtype=torch.float32, device=self.device)
        out = torch.empty(T, self.H, dtype=torch.bfloat16, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_shared_ffn_int8(self._h, xq.data_ptr(), x_scale.data_ptr(), T, self.packed.data_ptr(),
                                                hs.data_ptr(), hq.data_ptr(), sc.data_ptr(), out.data_ptr(), self._stream()))
        return out

    # ------------------------------------------------------------------ low-rank adapters
    def _plan_buffer(self, rows: int, n_adapters: int) -> torch.Tensor:
        return torch.empty_strided((_plan_bytes(rows, n_adapters),), (1,), dtype=torch.uint8, device=self.device)

    def adapter_plan(self, ids: torch.Tensor, n_adapters: int) -> AdapterPlan:
        """The rows of a batch sorted by adapter: ids [rows] int32, an id outside [0, n_adapters) for none."""
        self._check_in(ids, torch.int32, "ids")
        rows = ids.numel()
        buf = self._plan_buffer(rows, n_adapters)
        with self._on_device():
            L.check(self.lib.mg_adapter_plan(self._h, ids.data_ptr(), rows, n_adapters, buf.data_ptr(), self._stream()))
        return AdapterPlan(buf, rows, n_adapters)

    def adapter_plan_sorted(self, counts: torch.Tensor, pad_offsets: torch.Tensor, rows: int) -> AdapterPlan:
        """The plan of expert-sorted rows (permute_plan's counts and pad_offsets, buffers of `rows` rows), an adapter to an expert.  Rows in
        no expert's segment have none, those in front of the first offset among them."""
        self._check_in(counts, torch.int32, "counts")
        self._check_in(pad_offsets, torch.int32, "pad_offsets")
        n = counts.numel()
        if pad_offsets.numel() != n + 1:
            raise ValueError(f"counts of {n} and pad_offsets of {pad_offsets.numel()} entries")
        buf = self._plan_buffer(rows, n)
        with self._on_device():
            L.check(self.lib.mg_adapter_plan_sorted(self._h, counts.data_ptr(), pad_offsets.data_ptr(), rows, n, buf.data_ptr(),
                                                    self._stream()))
        return AdapterPlan(buf, rows, n)

    def _adapters(self, down: torch.Tensor, up: torch.Tensor, scale):
        """-> (mg_adapters as bytes, adapters, rank, cols, n_out, what the bytes point to)"""
        for t, what in ((down, "down"), (up, "up")):
            if t.dtype != torch.bfloat16 or t.dim() != 3 or t.device != self.device:
                raise ValueError(f"{what}: expected [adapters, rows, cols] bfloat16 on {self.device}, got {tuple(t.shape)} {t.dtype} on "
                                 f"{t.device}")
        n, rank, cols = down.shape
        n_up, n_out, rank_up = up.shape
        if n_up != n or rank_up != rank:
            raise ValueError(f"down {tuple(down.shape)} and up {tuple(up.shape)}")
        (sd, ld, one), (su, lu, one_up) = down.stride(), up.stride()
        if (cols > 1 and one != 1) or (rank > 1 and one_up != 1):
            raise ValueError(f"the elements of an adapter's row must be adjacent (strides {down.stride()}, {up.stride()})")
        factor, d_scale = 1.0, None
        if isinstance(scale, torch.Tensor):
            self._check_in(scale, torch.float32, "scale")
            if scale.numel() != n:
                raise ValueError(f"{scale.numel()} scales for {n} adapters")
            d_scale = scale.data_ptr()
        else:
            factor = float(scale)
        # torch leaves the strides of single rows open
        p_down, p_up = down.data_ptr(), up.data_ptr()
        ld, lu = ld if rank > 1 else (cols + 7) // 8 * 8, lu if n_out > 1 else (rank + 7) // 8 * 8
        if (p_down % 16 or ld % 8 or (n > 1 and sd % 8)) and down.is_contiguous():
            down = self._rows_on_boundaries(down)
            p_down, (sd, ld, _) = down.data_ptr(), down.stride()
        if (p_up % 16 or lu % 8 or (n > 1 and su % 8)) and up.is_contiguous():
            up = self._rows_on_boundaries(up)
            p_up, (su, lu, _) = up.data_ptr(), up.stride()
        return L.ADAPTERS.pack(L.ADAPTERS.size, n, rank, factor, cols, n_out, p_down, sd, ld, p_up, su, lu, d_scale or 0), n, rank, cols, n_out, \
            (down, up)

    def _rows_on_boundaries(self, t: torch.Tensor) -> torch.Tensor:
        """A copy of [matrices, rows, cols] bf16 whose rows begin on 16-byte boundaries."""
        n, rows, cols = t.shape
        ld = (cols + 7) // 8 * 8
        return torch.empty_strided((n, rows, cols), (rows * ld, ld, 1), dtype=torch.bfloat16, device=self.device).copy_(t.detach())

    def _adapter_plan_of(self, who, rows: int, n_adapters: int):
        """ids or a plan -> the two pointers of the call (what the ids lie in is the caller's)."""
        if isinstance(who, AdapterPlan):
            if who.rows != rows or who.n_adapters != n_adapters or who.buf.device != self.device:
                raise ValueError(f"plan of {who.rows} rows and {who.n_adapters} adapters on {who.buf.device} for {rows} and {n_adapters}")
            return who
        self._check_in(who, torch.int32, "ids")
        if who.numel() != rows:
            raise ValueError(f"{who.numel()} ids for {rows} rows")
        return who if rows <= L.ADAPTER_DIRECT else self.adapter_plan(who, n_adapters)

    def _rank_rows(self, rows: int, rank: int) -> torch.Tensor:
        n = _rank_stride(rank)
        return torch.empty_strided((rows, n), (n, 1), dtype=torch.bfloat16, device=self.device)

    def adapter_add(self, y: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, who, scale=1.0,
                    out: Optional[torch.Tensor] = None, keep: bool = False):
        """out[t] = y[t] + scale[g] * (x[t] . down[g]^T) . up[g]^T, g being row t's adapter; out[t] = y[t] for a row without one.
        x [rows, cols] and y [rows, n_out], down [adapters, rank, cols] and up [adapters, n_out, rank], bf16 with rows on 16-byte
        boundaries (views will do; contiguous adapters that lie otherwise are copied to such rows first, by every call); rank at most
        128, a lower one filled up with zeros.  who: int32 ids [rows], outside [0, adapters)
        for none, or the plan made of them (adapter_plan, adapter_plan_sorted), once for all of a batch's projections.  scale: a number or
        fp32 [adapters].  out may be y, and overlaps nothing otherwise.  With keep also the rows between the two products, in two
        parts of bf16, for adapter_grad: (out, s).  Any layer serves."""
        n, cols, ldx = self._rows_of(x, torch.bfloat16, "x")
        ad, n_adapters, rank, a_cols, a_out, _held = self._adapters(down, up, scale)
        if cols != a_cols:
            raise ValueError(f"down {tuple(down.shape)} for rows of {cols}")
        ny, n_out, ldy = self._rows_of(y, torch.bfloat16, "y")
        if (ny, n_out) != (n, a_out):
            raise ValueError(f"y {tuple(y.shape)}, expected {(n, a_out)}")
        who = self._adapter_plan_of(who, n, n_adapters)
        ids, plan = (None, who.buf) if isinstance(who, AdapterPlan) else (who, None)
        out, ldo = self._out_rows(out, n, n_out, "out", y, ldy)
        s = self._rank_rows(n, rank) if keep else None
        with self._on_device():
            L.check(self.lib.mg_adapter_add(self._h, ad, x.data_ptr(), ldx, y.data_ptr(), ldy, n, _ptr(ids), _ptr(plan),
                                            out.data_ptr(), ldo, _ptr(s), self._stream()))
        return (out, s) if keep else out

    def adapter_grad(self, grad_out: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, who, scale, s: torch.Tensor,
                     need_x: bool = True, need_down: bool = True, need_up: bool = True):
        """Gradients of adapter_add -> (grad_x, grad_down, grad_up), bf16, None for what is not needed; s is what adapter_add kept.
        grad_x is zero in rows without an adapter, the others in adapters without rows.  The gradient of y is grad_out itself."""
        n, cols, ldx = self._rows_of(x, torch.bfloat16, "x")
        ad, n_adapters, rank, a_cols, a_out, _held = self._adapters(down, up, scale)
        if cols != a_cols:
            raise ValueError(f"down {tuple(down.shape)} for rows of {cols}")
        ng, n_out, ldg = self._rows_of(grad_out, torch.bfloat16, "grad_out")
        if (ng, n_out) != (n, a_out):
            raise ValueError(f"grad_out {tuple(grad_out.shape)}, expected {(n, a_out)}")
        if isinstance(who, torch.Tensor):
            self._check_in(who, torch.int32, "ids")
            if who.numel() != n:
                raise ValueError(f"{who.numel()} ids for {n} rows")
            who = self.adapter_plan(who, n_adapters)
        who = self._adapter_plan_of(who, n, n_adapters)
        gs = self._rank_rows(n, rank)
        self._check_rows(s, torch.bfloat16, n, gs.shape[1], "s")
        if not (need_x or need_down or need_up):
            return None, None, None
        gx, ldgx = self._out_rows(None, n, cols, "grad_x", x, ldx) if need_x else (None, 0)
        gdown = torch.empty_like(down, memory_format=torch.contiguous_format) if need_down else None
        gup = torch.empty_like(up, memory_format=torch.contiguous_format) if need_up else None
        with self._on_device():
            L.check(self.lib.mg_adapter_grad(self._h, ad, grad_out.data_ptr(), ldg, x.data_ptr(), ldx, n, who.buf.data_ptr(),
                                             s.data_ptr(), gs.data_ptr(), _ptr(gx), ldgx, _ptr(gdown), _ptr(gup), self._stream()))
        return gx, gdown, gup

    @contextlib.contextmanager
    def job_counters(self, buf: torch.Tensor):
        """The expert calls inside hand out their jobs by counters in buf (int32 [JOB_COUNTERS] on the layer's
        device, theirs alone until they have run) instead of in fixed turns (mg_set_job_counters)."""
        self._check_in(buf, torch.int32, "job counters")
        if buf.numel() < L.JOB_COUNTERS:
            raise ValueError(f"job counters: {buf.numel()} words, {L.JOB_COUNTERS} needed")
        L.check(self.lib.mg_set_job_counters(self._h, buf.data_ptr()))
        try:
            yield
        finally:
            L.check(self.lib.mg_set_job_counters(self._h, None))

    def expert_ffn(self, perm_x: torch.Tensor, pad_offsets: torch.Tensor, counts: torch.Tensor,
                   predequant: bool = False):
        """-> (h_buf [rows,I], out_rows [rows,H]) over the padded expert-sorted rows.
        predequant=True (FP8 layers) de-quantises the weights into scratch first."""
        self._check_rows(perm_x, torch.bfloat16, None, self.H, "perm_x")
        self._check_in(counts, torch.int32, "counts")
        self._check_in(pad_offsets, torch.int32, "pad_offsets")
        if counts.numel() != self.e_local or pad_offsets.numel() != self.e_local + 1:
            raise ValueError(f"counts of {counts.numel()} and pad_offsets of {pad_offsets.numel()} entries for {self.e_local} experts")
        rows = perm_x.shape[0]
        hbuf = torch.zeros(rows, self.I, dtype=torch.bfloat16, device=self.device)
        out = torch.zeros(rows, self.H, dtype=torch.bfloat16, device=self.device)
        nb = C.c_size_t()
        L.check(self.lib.mg_dequant_ws_bytes(self._h, C.byref(nb)))
        deq = torch.empty(nb.value, dtype=torch.uint8, device=self.device) if (nb.value and predequant) else None
        with self._on_device():
            L.check(self.lib.mg_expert_ffn(self._h, perm_x.data_ptr(), pad_offsets.data_ptr(), counts.data_ptr(),
                                           rows, self.packed.data_ptr(), hbuf.data_ptr(), out.data_ptr(),
                                           _ptr(deq), self._stream()))
            if deq is not None:
                torch.cuda.current_stream().synchronize()
        return hbuf, out

    def shared_ffn(self, x: torch.Tensor) -> torch.Tensor:
        self._check_rows(x, torch.bfloat16, None, self.H, "hidden_states")
        T = x.shape[0]
        hs = torch.empty(T, self.Is, dtype=torch.bfloat16, device=self.device)
        out = torch.empty(T, self.H, dtype=torch.bfloat16, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_shared_ffn(self._h, x.data_ptr(), T, self.packed.data_ptr(), hs.data_ptr(),
                                           out.data_ptr(), self._stream()))
        return out

    def combine(self, out_rows: torch.Tensor, dst_row: torch.Tensor, topk_idx: torch.Tensor,
                topk_w: torch.Tensor, shared_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y[t] = sum_j topk_w[t, j] * out_rows[dst_row[t, j]] (+ shared_out[t]) in the layer's combine mode: rows in bf16, the plan and
        the picks in int32, weights in fp32.  Entries of dst_row that are negative or not below out_rows' rows are left out."""
        T = topk_idx.shape[0]
        self._check_rows(out_rows, torch.bfloat16, None, self.H, "out_rows")
        self._check_rows(dst_row, torch.int32, T, self.k, "dst_row")
        self._check_rows(topk_idx, torch.int32, T, self.k, "topk_idx")
        self._check_rows(topk_w, torch.float32, T, self.k, "topk_w")
        if shared_out is not None:
            self._check_rows(shared_out, torch.bfloat16, T, self.H, "shared_out")
        y = torch.empty(T, self.H, dtype=torch.bfloat16, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_combine_bounded(self._h, out_rows.data_ptr(), out_rows.shape[0], dst_row.data_ptr(),
                                                topk_idx.data_ptr(), topk_w.data_ptr(), _ptr(shared_out), T, y.data_ptr(),
                                                self._stream()))
        return y

    def dequant_fp8(self, q: torch.Tensor, scale_inv: torch.Tensor) -> torch.Tensor:
        """bf16(float(q) * scale[r/128][c/128]) (moe_gen/models/Wrapper.py:109-138)."""
        q = _whole(q.to(self.device))
        s = scale_inv.to(self.device, torch.float32).contiguous()
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=self.device)
        with self._on_device():
            L.check(self.lib.mg_dequant_fp8_block128(q.data_ptr(), s.data_ptr(), q.shape[0], q.shape[1],
                                                     out.data_ptr(), self._stream()))
        return out
