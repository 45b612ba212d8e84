"""Torch-facing wrappers of the single-kernel C-ABI entry points.

Each wrapper validates device, dtype, contiguity and shape the way the
reference's custom op does (v16_1_clean.py:323-335: TypeError/ValueError on
bad inputs), then passes raw pointers and the current CUDA stream to the
library.  They exist for the per-kernel parity tests and for callers that
compose the layer themselves; UserOptimizedTransformer uses the single
tj_encoder_forward entry point.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib


def _stream(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def head_pad(head_dim: int) -> int:
    """Row length (halves) of the head-major q/k/v buffers: heads are
    zero-padded to 64, 128 or 256."""
    if not 1 <= head_dim <= 256:
        raise ValueError(f"head_dim must be in 1..256, got {head_dim}")
    return 64 if head_dim <= 64 else (128 if head_dim <= 128 else 256)


def _require(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _require_out(out: torch.Tensor, name: str, shape, dtype: torch.dtype, device: torch.device) -> None:
    """A caller-provided output must be exactly the buffer the kernel writes:
    the C ABI takes raw pointers and cannot check sizes itself."""
    _require(out, name, dtype, device)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(out.shape)}")


def token_plan(mask: Optional[torch.Tensor], batch: int, seq_len: int, device) -> torch.Tensor:
    lib = _lib.load()
    n = lib.tj_token_plan_ints(batch, seq_len)
    plan = torch.empty(n, dtype=torch.int32, device=device)
    mptr = None
    if mask is not None:
        if mask.shape != (batch, seq_len):
            raise ValueError(f"mask must be [{batch}, {seq_len}], got {tuple(mask.shape)}")
        m = mask.contiguous()
        if m.dtype == torch.bool:
            m = m.view(torch.uint8)
        _require(m, "mask", torch.uint8, plan.device)
        mptr = m.data_ptr()
    _lib.check(lib.tj_token_plan(mptr, batch, seq_len, plan.data_ptr(), _stream(plan)), "token_plan")
    return plan


def plan_views(plan: torch.Tensor, batch: int, seq_len: int):
    """(nv[1], cu[B+1], counts[B], orig[BS], inv[BS]) views of a token plan (it
    ends with order[B], the samples by decreasing count: plan_order)."""
    B, BS = batch, batch * seq_len
    nv = plan[0:1]
    cu = plan[1 : B + 2]
    cnt = plan[B + 2 : 2 * B + 2]
    orig = plan[2 * B + 2 : 2 * B + 2 + BS]
    inv = plan[2 * B + 2 + BS : 2 * B + 2 + 2 * BS]
    return nv, cu, cnt, orig, inv


def plan_order(plan: torch.Tensor, batch: int, seq_len: int) -> torch.Tensor:
    """order[B] of a token plan: samples by decreasing valid count (stable;
    the identity for batches above 256)."""
    off = 2 * batch + 2 + 2 * batch * seq_len
    return plan[off : off + batch]


def ln_cast_f16(x, gamma, beta, eps=1e-5, row_map=None, row_count=None, out=None):
    dev = x.device
    _require(x, "x", torch.float32, dev)
    D = x.shape[-1]
    rows = x.numel() // D if row_map is None else row_map.numel()
    if out is None:
        out = torch.empty(rows, D, dtype=torch.float16, device=dev)
    if out.dim() != 2 or out.shape[1] != D or out.shape[0] < rows:
        raise ValueError(f"out must be [>= {rows}, {D}], got {tuple(out.shape)}")
    _require(out, "out", torch.float16, dev)
    lib = _lib.load()
    rc = lib.tj_ln_cast_f16(
        x.data_ptr(), _ptr(row_map), _ptr(row_count), rows, D, gamma.data_ptr(), beta.data_ptr(),
        float(eps), out.data_ptr(), _stream(x),
    )
    _lib.check(rc, "ln_cast_f16")
    return out


def ln_final_mask(x, gamma, beta, eps=1e-5, inv_map=None, rows=None, out=None):
    dev = x.device
    _require(x, "x", torch.float32, dev)
    D = x.shape[-1]
    if rows is None:
        rows = x.numel() // D if inv_map is None else inv_map.numel()
    if out is None:
        out = torch.empty(rows, D, dtype=torch.float32, device=dev)
    _require_out(out, "out", (rows, D), torch.float32, dev)
    lib = _lib.load()
    rc = lib.tj_ln_final_mask(
        x.data_ptr(), _ptr(inv_map), rows, D, gamma.data_ptr(), beta.data_ptr(), float(eps),
        out.data_ptr(), _stream(x),
    )
    _lib.check(rc, "ln_final_mask")
    return out


def add_ln_cast_f16(x, add16, gamma, beta, eps=1e-5, row_map=None, row_count=None, sum_out=None,
                    out=None):
    """s = x[row_map[r]] + add16[r] (fp32); sum_out[r] = s; out[r] = fp16(LayerNorm(s))."""
    dev = x.device
    _require(x, "x", torch.float32, dev)
    _require(add16, "add16", torch.float16, dev)
    D = x.shape[-1]
    rows = x.numel() // D if row_map is None else row_map.numel()
    if add16.dim() != 2 or add16.shape[1] != D or add16.shape[0] < rows:
        raise ValueError(f"add16 must be [>= {rows}, {D}], got {tuple(add16.shape)}")
    if out is None:
        out = torch.empty(rows, D, dtype=torch.float16, device=dev)
    if out.dim() != 2 or out.shape[1] != D or out.shape[0] < rows:
        raise ValueError(f"out must be [>= {rows}, {D}], got {tuple(out.shape)}")
    _require(out, "out", torch.float16, dev)
    if sum_out is not None:
        _require(sum_out, "sum_out", torch.float32, dev)
        if sum_out.dim() != 2 or sum_out.shape[1] != D or sum_out.shape[0] < rows:
            raise ValueError(f"sum_out must be [>= {rows}, {D}], got {tuple(sum_out.shape)}")
    lib = _lib.load()
    rc = lib.tj_add_ln_cast_f16(
        x.data_ptr(), _ptr(row_map), add16.data_ptr(), _ptr(row_count), rows, D, gamma.data_ptr(),
        beta.data_ptr(), float(eps), _ptr(sum_out), out.data_ptr(), _stream(x),
    )
    _lib.check(rc, "add_ln_cast_f16")
    return out


def add_ln_final_mask(x, add16, gamma, beta, eps=1e-5, inv_map=None, rows=None, out=None):
    """out[m] = LayerNorm(x[c] + add16[c]), c = inv_map[m] (zeros where c < 0)."""
    dev = x.device
    _require(x, "x", torch.float32, dev)
    _require(add16, "add16", torch.float16, dev)
    D = x.shape[-1]
    if add16.shape != x.shape:
        raise ValueError(f"add16 must match x {tuple(x.shape)}, got {tuple(add16.shape)}")
    if rows is None:
        rows = x.numel() // D if inv_map is None else inv_map.numel()
    if out is None:
        out = torch.empty(rows, D, dtype=torch.float32, device=dev)
    _require_out(out, "out", (rows, D), torch.float32, dev)
    lib = _lib.load()
    rc = lib.tj_add_ln_final_mask(
        x.data_ptr(), add16.data_ptr(), _ptr(inv_map), rows, D, gamma.data_ptr(), beta.data_ptr(),
        float(eps), out.data_ptr(), _stream(x),
    )
    _lib.check(rc, "add_ln_final_mask")
    return out


def add2_ln_final_mask(x, attn16, ffn16, gamma, beta, eps=1e-5, inv_map=None, x_at_original=False,
                       rows=None, out=None):
    """out[m] = LayerNorm((x[r] + attn16[c]) + ffn16[c]), c = inv_map[m], r = m if
    x_at_original else c (zeros where c < 0)."""
    dev = x.device
    _require(x, "x", torch.float32, dev)
    _require(attn16, "attn16", torch.float16, dev)
    _require(ffn16, "ffn16", torch.float16, dev)
    D = x.shape[-1]
    if attn16.shape != ffn16.shape or attn16.dim() != 2 or attn16.shape[1] != D:
        raise ValueError("attn16 and ffn16 must both be [compact_rows, D]")
    if rows is None:
        rows = x.numel() // D if inv_map is None else inv_map.numel()
    if x_at_original and (inv_map is None or x.numel() // D < rows):
        raise ValueError("x_at_original needs inv_map and x holding every output row")
    if out is None:
        out = torch.empty(rows, D, dtype=torch.float32, device=dev)
    _require_out(out, "out", (rows, D), torch.float32, dev)
    lib = _lib.load()
    rc = lib.tj_add2_ln_final_mask(
        x.data_ptr(), 1 if x_at_original else 0, attn16.data_ptr(), ffn16.data_ptr(), _ptr(inv_map), rows,
        D, gamma.data_ptr(), beta.data_ptr(), float(eps), out.data_ptr(), _stream(x),
    )
    _lib.check(rc, "add2_ln_final_mask")
    return out


def gemm_qkv_headmajor(a16, w_qkv16, b_qkv, num_heads, row_count=None, out=None):
    dev = a16.device
    _require(a16, "a16", torch.float16, dev)
    _require(w_qkv16, "w_qkv16", torch.float16, dev)
    _require(b_qkv, "b_qkv", torch.float32, dev)
    rows, D = a16.shape
    if w_qkv16.shape != (3 * D, D):
        raise ValueError(f"w_qkv16 must be [{3 * D}, {D}], got {tuple(w_qkv16.shape)}")
    if out is None:
        # head-major, each head zero-padded to head_pad(D // H) halves
        out = torch.empty(3, num_heads, rows, head_pad(D // num_heads), dtype=torch.float16, device=dev)
    _require_out(out, "out", (3, num_heads, rows, head_pad(D // num_heads)), torch.float16, dev)
    lib = _lib.load()
    rc = lib.tj_gemm_qkv_headmajor(
        a16.data_ptr(), w_qkv16.data_ptr(), b_qkv.data_ptr(), _ptr(row_count), rows, D, num_heads,
        out.data_ptr(), _stream(a16),
    )
    _lib.check(rc, "gemm_qkv_headmajor")
    return out


def gemm_bias_residual_f32(a16, w16, bias, resid, resid_map=None, row_count=None, out=None):
    dev = a16.device
    _require(a16, "a16", torch.float16, dev)
    _require(w16, "w16", torch.float16, dev)
    _require(bias, "bias", torch.float32, dev)
    _require(resid, "resid", torch.float32, dev)
    rows, K = a16.shape
    N = w16.shape[0]
    if w16.shape[1] != K:
        raise ValueError("w16 inner dimension does not match a16")
    if out is None:
        out = torch.empty(rows, N, dtype=torch.float32, device=dev)
    if out.dim() != 2 or out.shape[1] != N or out.shape[0] < (rows if row_count is None else 1):
        raise ValueError(f"out must be [rows, {N}], got {tuple(out.shape)}")
    _require(out, "out", torch.float32, dev)
    if resid.dim() != 2 or resid.shape[1] != N:
        raise ValueError(f"resid must be [rows, {N}], got {tuple(resid.shape)}")
    if resid_map is None and row_count is None and resid.shape[0] < rows:
        raise ValueError("resid has fewer rows than a16")
    lib = _lib.load()
    rc = lib.tj_gemm_bias_residual_f32(
        a16.data_ptr(), w16.data_ptr(), bias.data_ptr(), resid.data_ptr(), _ptr(resid_map),
        _ptr(row_count), rows, N, K, out.data_ptr(), _stream(a16),
    )
    _lib.check(rc, "gemm_bias_residual_f32")
    return out


def gemm_bias_f16(a16, w16, bias, row_count=None, out=None):
    """fp16 out = a16 @ w16^T + bias (the reference's fp16 F.linear)."""
    dev = a16.device
    _require(a16, "a16", torch.float16, dev)
    _require(w16, "w16", torch.float16, dev)
    _require(bias, "bias", torch.float32, dev)
    rows, K = a16.shape
    N = w16.shape[0]
    if w16.shape[1] != K:
        raise ValueError("w16 inner dimension does not match a16")
    if out is None:
        out = torch.empty(rows, N, dtype=torch.float16, device=dev)
    _require_out(out, "out", (rows, N), torch.float16, dev)
    lib = _lib.load()
    rc = lib.tj_gemm_bias_f16(
        a16.data_ptr(), w16.data_ptr(), bias.data_ptr(), _ptr(row_count), rows, N, K, out.data_ptr(),
        _stream(a16),
    )
    _lib.check(rc, "gemm_bias_f16")
    return out


def gemm_bias_gelu_f16(a16, w16, bias, row_count=None, out=None):
    dev = a16.device
    _require(a16, "a16", torch.float16, dev)
    _require(w16, "w16", torch.float16, dev)
    _require(bias, "bias", torch.float32, dev)
    rows, K = a16.shape
    N = w16.shape[0]
    if w16.shape[1] != K:
        raise ValueError("w16 inner dimension does not match a16")
    if out is None:
        out = torch.empty(rows, N, dtype=torch.float16, device=dev)
    _require_out(out, "out", (rows, N), torch.float16, dev)
    lib = _lib.load()
    rc = lib.tj_gemm_bias_gelu_f16(
        a16.data_ptr(), w16.data_ptr(), bias.data_ptr(), _ptr(row_count), rows, N, K,
        out.data_ptr(), _stream(a16),
    )
    _lib.check(rc, "gemm_bias_gelu_f16")
    return out


def flash_attn_fwd(q, k, v, q_cu, kv_off, kv_len, max_q_per_sample, scale, causal=False,
                   q_pos0=None, out=None, head_dim=64, part_o=None, part_lse=None, part_mode=0):
    """q: [H, q_rows, P]; k, v: [G, H, kv_rows, P] with P = head_pad(head_dim) (any strides
    with unit inner stride; rows hold head_dim values then zeros up to P); q_cu: [B+1];
    kv_off/kv_len: [B, G]
    int32.  Returns ctx [q_rows, H*head_dim] fp16.

    Split attention (tj_flash_attn_fwd_partial): part_mode 1 writes the partial
    result of these keys into part_o [q_rows, H*head_dim] fp32 and part_lse
    [q_rows, H] fp32 and returns None; part_mode 2 merges these keys with that
    partial into ctx."""
    dev = q.device
    _require(q, "q", torch.float16, dev)
    if k.dim() == 3:
        k = k.unsqueeze(0)
        v = v.unsqueeze(0)
    G, H, kv_rows, row = k.shape
    dh = head_dim
    P = head_pad(dh)
    if row != P or q.shape[0] != H or q.shape[2] != P:
        raise ValueError(f"q, k, v rows must be {P} halves (head dim {dh} zero-padded)")
    if k.stride() != v.stride() or k.stride(-1) != 1 or k.stride(-2) != P:
        raise ValueError(f"k and v must share strides with contiguous [rows, {P}] slabs")
    B = q_cu.numel() - 1
    if part_mode not in (0, 1, 2):
        raise ValueError(f"part_mode must be 0, 1 or 2, got {part_mode}")
    if part_mode:
        _require_out(part_o, "part_o", (q.shape[1], H * dh), torch.float32, dev)
        _require_out(part_lse, "part_lse", (q.shape[1], H), torch.float32, dev)
    if part_mode == 1:
        out = None
    elif out is None:
        out = torch.empty(q.shape[1], H * dh, dtype=torch.float16, device=dev)
    # out may be a column slice of a wider context (a head group's columns):
    # rows of H*head_dim contiguous halves at any row stride.
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.dtype != torch.float16 or out.device != dev:
            raise TypeError(f"out must be a float16 tensor on {dev}")
        if tuple(out.shape) != (q.shape[1], H * dh) or out.stride(1) != 1 or out.stride(0) < H * dh:
            raise ValueError(f"out must be [{q.shape[1]}, {H * dh}] with contiguous rows, got "
                             f"{tuple(out.shape)} strides {out.stride()}")
    for name, t in (("q_cu", q_cu), ("kv_off", kv_off), ("kv_len", kv_len)):
        _require(t, name, torch.int32, dev)
    if kv_off.numel() != B * G or kv_len.numel() != B * G:
        raise ValueError(f"kv_off/kv_len must hold {B}x{G} entries")
    lib = _lib.load()
    rc = lib.tj_flash_attn_fwd_partial(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), H, dh, q.shape[1], kv_rows, k.stride(1),
        k.stride(0), G, B, max_q_per_sample, q_cu.data_ptr(), kv_off.data_ptr(),
        kv_len.data_ptr(), float(scale), 1 if causal else 0, _ptr(q_pos0), _ptr(out),
        0 if out is None else out.stride(0), _ptr(part_o), _ptr(part_lse), part_mode, _stream(q),
    )
    _lib.check(rc, "flash_attn_fwd")
    return out


# ---- expert feed-forward ------------------------------------------------------
# A call on one token is bound by the host, so these wrappers make few torch
# calls: no device guard where the device is current, the raw stream handle.
def _launch(dev: torch.device, fn, *args) -> int:
    """fn(*args, stream) with dev current, on dev's current stream."""
    if torch.cuda.current_device() == dev.index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    with torch.cuda.device(dev):
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))


_DTYPES = {torch.float32: _lib.TJ_DTYPE_F32, torch.float16: _lib.TJ_DTYPE_F16, torch.bfloat16: _lib.TJ_DTYPE_BF16}
_SCORES = {"softmax": _lib.TJ_SCORE_SOFTMAX, "sigmoid": _lib.TJ_SCORE_SIGMOID}
_GATES = {"none": _lib.TJ_GATE_NONE, "sigmoid": _lib.TJ_GATE_SIGMOID, "tanh": _lib.TJ_GATE_TANH}


def _no_grad(*tensors) -> None:
    """Forward only, like the encoder: a call whose gradient (or forward-mode
    tangent, which no_grad does not switch off) would be lost raises."""
    if forward_ad._current_level >= 0:  # inside a dual_level
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("forward-mode autograd through this operator is not supported")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("autograd through this operator is not supported; call it under torch.no_grad()")


def _cuda_tensor(t, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (the library has no CPU path)")
    return t.device


def _require_shape(t, name: str, shape, dtype: torch.dtype, device: torch.device) -> None:
    if isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == dtype and t.device == device and t.is_contiguous():
        return
    _require(t, name, dtype, device)
    raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _require_ints(**values) -> None:
    """The C entries take 32-bit ints, and ctypes would drop the rest without a word."""
    for name, v in values.items():
        if not -(2**31) <= v < 2**31:
            raise ValueError(f"{name} = {v} does not fit 32 bits")


def _require_count(row_count, device: torch.device) -> None:
    if row_count is not None:
        _require(row_count, "row_count", torch.int32, device)
        if row_count.numel() != 1:
            raise ValueError("row_count must hold one int32")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share bytes."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    return (a.data_ptr() < b.data_ptr() + b.numel() * b.element_size()
            and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())


def _require_apart(out: torch.Tensor, name: str, **others) -> None:
    """out shares no memory with an input that the kernels may read after its first rows are written."""
    for other, t in others.items():
        if t is not None and _overlap(out, t):
            raise ValueError(f"{name} must not share memory with {other}")


def _half_dtype(t: torch.Tensor, name: str) -> int:
    if t.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{name} must be float16 or bfloat16, got {t.dtype}")
    return _DTYPES[t.dtype]


@dataclass
class ExpertRouting:
    """Choices of a batch of rows and the plan the expert kernels read: `experts`
    [rows, top_k] int32 (-1: none), `weights` [rows, top_k] float32, and
    `plan`, whose parts are the properties below.  Slots are the (row, j)
    pairs sorted by expert, in (row, j) order inside an expert.  `row_count`
    is the device int given to the router (None: all rows)."""

    experts: torch.Tensor
    weights: torch.Tensor
    plan: torch.Tensor
    num_experts: int
    row_count: Optional[torch.Tensor] = None

    def __post_init__(self) -> None:
        # the kernels take these buffers by pointer
        if self.experts.dim() != 2:
            raise ValueError(f"experts must be [rows, top_k], got {tuple(self.experts.shape)}")
        dev = self.plan.device
        _require(self.experts, "experts", torch.int32, dev)
        _require_ints(rows=self.experts.shape[0], num_experts=self.num_experts)
        _require_shape(self.weights, "weights", self.experts.shape, torch.float32, dev)
        _require(self.plan, "plan", torch.int32, dev)
        if self.plan.numel() < self.num_experts + 1 + 2 * self.experts.numel():
            raise ValueError(f"plan of {self.plan.numel()} entries is too short for {tuple(self.experts.shape)} choices "
                             f"of {self.num_experts} experts")
        _require_count(self.row_count, dev)

    @classmethod
    def _made(cls, experts, weights, plan, num_experts, row_count) -> "ExpertRouting":
        """From buffers made here, without the checks."""
        r = cls.__new__(cls)
        r.experts, r.weights, r.plan, r.num_experts, r.row_count = experts, weights, plan, num_experts, row_count
        return r

    @property
    def rows(self) -> int:
        return self.experts.shape[0]

    @property
    def top_k(self) -> int:
        return self.experts.shape[1]

    @property
    def offsets(self) -> torch.Tensor:
        """[num_experts + 1]: expert e has slots offsets[e] .. offsets[e+1]."""
        return self.plan[: self.num_experts + 1]

    @property
    def slot_row(self) -> torch.Tensor:
        """[rows * top_k]: row of each slot, -1 past the last slot."""
        n = self.num_experts + 1
        return self.plan[n : n + self.rows * self.top_k]

    @property
    def row_slot(self) -> torch.Tensor:
        """[rows, top_k]: slot of each choice, -1 without an expert."""
        n, s = self.num_experts + 1, self.rows * self.top_k
        return self.plan[n + s : n + 2 * s].view(self.rows, self.top_k)


def _plan_buffer(rows: int, top_k: int, num_experts: int, device: torch.device) -> torch.Tensor:
    n = _lib.load().tj_expert_plan_ints(rows, top_k, num_experts)
    return torch.empty(n, dtype=torch.int32, device=device)


def route_experts(logits, top_k, *, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_score_top=1,
                  renormalize=True, weight_scale=1.0, row_count=None) -> ExpertRouting:
    """Routes each row of logits [rows, E] (float32, float16 or bfloat16) to its
    top_k experts and sorts the choices by expert.

    Scores are the row's softmax or sigmoid; the experts with the greatest
    score + bias (bias: [E] float32) are chosen, as by 64-bit values, equal ones
    by their logits and then in index order, and with num_groups > 1 only among the top_groups groups with the greatest
    sum of their group_score_top (1 or 2) best values.  Weights are the scores
    of the chosen, divided by their sum if renormalize, times weight_scale.  A
    logit of -inf closes an expert to the row (a row without enough open
    experts ends in -1 with weight 0), a row with a NaN has NaN weights, and
    rows at or past row_count (a device int32) are not routed."""
    dev = _cuda_tensor(logits, "logits")
    _no_grad(logits, bias)
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    _require(logits, "logits", logits.dtype, dev)
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, experts], got {tuple(logits.shape)}")
    rows, E = logits.shape
    if rows >= 2**31 or num_groups != 1 or top_groups != 1 or group_score_top != 1:
        _require_ints(rows=rows, num_groups=num_groups, top_groups=top_groups, group_score_top=group_score_top)
    if scoring not in _SCORES:
        raise ValueError(f"scoring must be one of {sorted(_SCORES)}, got {scoring!r}")
    if not 1 <= top_k <= min(E, 32):
        raise ValueError(f"top_k must be in 1..{min(E, 32)}, got {top_k}")
    if bias is not None:
        _require_shape(bias, "bias", (E,), torch.float32, dev)
    _require_count(row_count, dev)
    lib = _lib.load()
    experts = torch.empty(rows, top_k, dtype=torch.int32, device=dev)
    weights = torch.empty(rows, top_k, dtype=torch.float32, device=dev)
    plan = _plan_buffer(rows, top_k, E, dev)
    rc = _launch(
        dev, lib.tj_route_experts, logits.data_ptr(), _DTYPES[logits.dtype], rows, _ptr(row_count), E, top_k,
        _SCORES[scoring], _ptr(bias), num_groups, top_groups, group_score_top, 1 if renormalize else 0, weight_scale,
        experts.data_ptr(), weights.data_ptr(), plan.data_ptr(),
    )
    _lib.check(rc, "route_experts")
    return ExpertRouting._made(experts, weights, plan, E, row_count)


def expert_plan(experts, weights, num_experts, *, row_count=None) -> ExpertRouting:
    """Routing made of choices from elsewhere: experts [rows, top_k] int32
    (negative: none; a row may name an expert twice) and weights [rows, top_k]
    float32.  An index >= num_experts is a device error and counts as none."""
    dev = _cuda_tensor(experts, "experts")
    _no_grad(weights)
    _require(experts, "experts", torch.int32, dev)
    if experts.dim() != 2 or not 1 <= experts.shape[1] <= 32:
        raise ValueError(f"experts must be [rows, top_k] with top_k in 1..32, got {tuple(experts.shape)}")
    rows, top_k = experts.shape
    _require_ints(rows=rows)
    _require_shape(weights, "weights", (rows, top_k), torch.float32, dev)
    _require_count(row_count, dev)
    if not 1 <= num_experts <= 512:
        raise ValueError(f"num_experts must be in 1..512, got {num_experts}")
    plan = _plan_buffer(rows, top_k, num_experts, dev)
    rc = _launch(dev, _lib.load().tj_expert_plan, experts.data_ptr(), rows, top_k, _ptr(row_count), num_experts,
                 plan.data_ptr())
    _lib.check(rc, "expert_plan")
    return ExpertRouting._made(experts, weights, plan, num_experts, row_count)


def _require_routing(routing, device: torch.device) -> None:
    if not isinstance(routing, ExpertRouting):
        raise TypeError("routing must be an ExpertRouting (route_experts, expert_plan)")
    if routing.plan.device != device:
        raise ValueError(f"routing must be on {device}, got {routing.plan.device}")


def gemm_experts(a, w, bias, routing, *, gather, gelu=False, out=None):
    """out[s] = act(w[e] @ a[r] + bias[e]) for every slot s of the routing, e its
    expert and r its row (gather: a is [rows, K]) or s (a is [rows * top_k, K]);
    act is erf-GELU or none.  w [E, N, K], bias [E, N] float32 or None, N and K
    multiples of 8.  Rows of out [rows * top_k, N] past the last slot are left
    as they were."""
    dev = _cuda_tensor(a, "a")
    _no_grad(a, w, bias)
    code = _half_dtype(a, "a")
    _require_routing(routing, dev)
    slots = routing.rows * routing.top_k
    if a.dim() != 2:
        raise ValueError(f"a must be a matrix, got {tuple(a.shape)}")
    K = a.shape[1]
    _require_shape(a, "a", (routing.rows if gather else slots, K), a.dtype, dev)
    _require(w, "w", a.dtype, dev)
    if w.dim() != 3 or w.shape[0] != routing.num_experts or w.shape[2] != K:
        raise ValueError(f"w must be [{routing.num_experts}, N, {K}], got {tuple(w.shape)}")
    N = w.shape[1]
    if N >= 2**31 or K >= 2**31:
        _require_ints(N=N, K=K)
    if bias is not None:
        _require_shape(bias, "bias", (routing.num_experts, N), torch.float32, dev)
    if out is None:
        out = torch.empty(slots, N, dtype=a.dtype, device=dev)
    else:
        _require_out(out, "out", (slots, N), a.dtype, dev)
        _require_apart(out, "out", a=a, w=w, bias=bias, routing=routing.plan)
    lib = _lib.load()
    need = lib.tj_gemm_experts_workspace_bytes(routing.rows, routing.top_k, routing.num_experts, K, 1 if gather else 0)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    rc = _launch(
        dev, lib.tj_gemm_experts, a.data_ptr(), code, 1 if gather else 0, w.data_ptr(), _ptr(bias),
        routing.plan.data_ptr(), routing.rows, routing.top_k, routing.num_experts, N, K, 1 if gelu else 0,
        out.data_ptr(), _ptr(ws), need,
    )
    _lib.check(rc, "gemm_experts")
    return out


def expert_combine(y, routing, *, out=None):
    """out[r] = sum_j weights[r, j] * y[slot(r, j)], zeros for a row without
    experts; rows at or past the routing's row_count are left as they were."""
    dev = _cuda_tensor(y, "y")
    _no_grad(y, routing.weights if isinstance(routing, ExpertRouting) else None)
    code = _half_dtype(y, "y")
    _require_routing(routing, dev)
    if y.dim() != 2:
        raise ValueError(f"y must be a matrix, got {tuple(y.shape)}")
    D = y.shape[1]
    _require_shape(y, "y", (routing.rows * routing.top_k, D), y.dtype, dev)
    _require_ints(D=D)
    if out is None:
        out = torch.empty(routing.rows, D, dtype=y.dtype, device=dev)
    else:
        _require_out(out, "out", (routing.rows, D), y.dtype, dev)
        _require_apart(out, "out", y=y, weights=routing.weights, routing=routing.plan, row_count=routing.row_count)
    rc = _launch(
        dev, _lib.load().tj_expert_combine, y.data_ptr(), code, routing.weights.data_ptr(), routing.plan.data_ptr(),
        _ptr(routing.row_count), routing.rows, routing.top_k, routing.num_experts, D, out.data_ptr(),
    )
    _lib.check(rc, "expert_combine")
    return out


def expert_ffn(a, w_in, b_in, w_out, b_out, routing, *, out=None):
    """The routed feed-forward of a [rows, D] (float16 or bfloat16): each row's
    experts run ffn_in, erf-GELU and ffn_out on it and out is their weighted
    sum.  w_in [E, F, D], w_out [E, D, F], biases [E, F] and [E, D] float32 or
    None, D and F multiples of 8.  Zeros for a row without experts; rows at or
    past the routing's row_count are left as they were.  out may be a."""
    dev = _cuda_tensor(a, "a")
    _no_grad(a, w_in, b_in, w_out, b_out)
    code = _half_dtype(a, "a")
    _require_routing(routing, dev)
    _no_grad(routing.weights)
    E = routing.num_experts
    if a.dim() != 2 or a.shape[0] != routing.rows:
        raise ValueError(f"a must be [{routing.rows}, D], got {tuple(a.shape)}")
    _require(a, "a", a.dtype, dev)
    D = a.shape[1]
    _require(w_in, "w_in", a.dtype, dev)
    if w_in.dim() != 3 or w_in.shape[0] != E or w_in.shape[2] != D:
        raise ValueError(f"w_in must be [{E}, F, {D}], got {tuple(w_in.shape)}")
    F = w_in.shape[1]
    if D >= 2**31 or F >= 2**31:
        _require_ints(D=D, F=F)
    _require_shape(w_out, "w_out", (E, D, F), a.dtype, dev)
    if b_in is not None:
        _require_shape(b_in, "b_in", (E, F), torch.float32, dev)
    if b_out is not None:
        _require_shape(b_out, "b_out", (E, D), torch.float32, dev)
    rows, top_k = routing.experts.shape
    if out is None:
        out = torch.empty(rows, D, dtype=a.dtype, device=dev)
    else:
        _require_out(out, "out", (rows, D), a.dtype, dev)
        _require_apart(out, "out", w_in=w_in, b_in=b_in, w_out=w_out, b_out=b_out, weights=routing.weights,
                       routing=routing.plan, row_count=routing.row_count)
    lib = _lib.load()
    need = lib.tj_expert_ffn_workspace_bytes(rows, top_k, E, D, F)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    rc = _launch(
        dev, lib.tj_expert_ffn, a.data_ptr(), code, w_in.data_ptr(), _ptr(b_in), w_out.data_ptr(), _ptr(b_out),
        routing.weights.data_ptr(), routing.plan.data_ptr(), _ptr(routing.row_count), rows, top_k, E, D, F,
        out.data_ptr(), ws.data_ptr(), need,
    )
    _lib.check(rc, "expert_ffn")
    return out


def sandwich_norm(x, branch, pre_gamma, pre_beta=None, *, post_gamma=None, post_beta=None, kind="layer", gate=None,
                  gate_act="none", rows_per_gate=1, gate_map=None, residual_scale=1.0, eps=1e-5, row_map=None,
                  row_count=None, routing=None, sum_out=None, out=None):
    """The residual step between two blocks, with a norm behind one and a norm
    before the next:

        s[r] = x[row_map[r]] + residual_scale * act(gate) * post(b[r])
        y[r] = pre(s[r])

    returning (s float32, y in branch's dtype).  b is branch [rows, D] (float16
    or bfloat16), or with `routing` the weighted sum of branch [rows * top_k,
    D], its experts' outputs in slot order.  post and pre are LayerNorm
    (kind="layer") or RMSNorm ("rms"); no post_gamma: no norm of the branch.
    gate: [D] (float32) per channel, or [G, D] (float32 or branch's dtype) with
    row r reading gate row gate_map[r] // rows_per_gate (gate_map: int32,
    default row_map, else r): a sample's gate with rows_per_gate = seq_len, a
    token's with 1.  act: none, sigmoid or tanh.  x [x_rows, D] float32; sum_out
    may be x when there is no row_map, out branch when there is no routing, and
    neither may share memory with another input.  Rows at or past row_count
    (default: the routing's) are left as they were."""
    dev = _cuda_tensor(x, "x")
    _no_grad(x, branch, pre_gamma, pre_beta, post_gamma, post_beta, gate)
    _require(x, "x", torch.float32, dev)
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, D], got {tuple(x.shape)}")
    D = x.shape[1]
    _cuda_tensor(branch, "branch")
    code = _half_dtype(branch, "branch")
    if kind not in ("layer", "rms"):
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    if gate_act not in _GATES:
        raise ValueError(f"gate_act must be one of {sorted(_GATES)}, got {gate_act!r}")
    if routing is not None:
        _require_routing(routing, dev)
        _no_grad(routing.weights)
        rows = routing.rows
        _require_shape(branch, "branch", (rows * routing.top_k, D), branch.dtype, dev)
        if row_count is None:
            row_count = routing.row_count
    else:
        if branch.dim() != 2:
            raise ValueError(f"branch must be [rows, {D}], got {tuple(branch.shape)}")
        rows = branch.shape[0]
        _require_shape(branch, "branch", (rows, D), branch.dtype, dev)
    if rows >= 2**31 or x.shape[0] >= 2**31 or D >= 2**31:
        _require_ints(rows=rows, x_rows=x.shape[0], columns=D)
    _require_count(row_count, dev)
    if row_map is not None:
        _require_shape(row_map, "row_map", (rows,), torch.int32, dev)
    elif x.shape[0] < rows:
        raise ValueError(f"x must have at least {rows} rows, got {x.shape[0]}")
    vector = (D,)
    if pre_gamma is None:
        raise ValueError("pre_gamma is required")
    _require_shape(pre_gamma, "pre_gamma", vector, torch.float32, dev)
    if pre_beta is not None:
        _require_shape(pre_beta, "pre_beta", vector, torch.float32, dev)
    if post_gamma is not None:
        _require_shape(post_gamma, "post_gamma", vector, torch.float32, dev)
    if post_beta is not None:
        _require_shape(post_beta, "post_beta", vector, torch.float32, dev)
    if post_beta is not None and post_gamma is None:
        raise ValueError("post_beta needs post_gamma")
    gate_rows, gate_code = 0, _lib.TJ_DTYPE_F32
    if gate is not None:
        if gate.dim() == 1:
            _require_shape(gate, "gate", (D,), torch.float32, dev)
            gate_rows, rows_per_gate, gate_map = 1, max(rows, 1), None
        else:
            if gate.dtype not in (torch.float32, branch.dtype):
                raise TypeError(f"gate must be float32 or {branch.dtype}, got {gate.dtype}")
            _require(gate, "gate", gate.dtype, dev)
            if gate.dim() != 2 or gate.shape[1] != D or gate.shape[0] < 1:
                raise ValueError(f"gate must be [{D}] or [G, {D}], got {tuple(gate.shape)}")
            if rows_per_gate < 1:
                raise ValueError(f"rows_per_gate must be at least 1, got {rows_per_gate}")
            gate_rows, gate_code = gate.shape[0], _DTYPES[gate.dtype]
            _require_ints(gate_rows=gate_rows, rows_per_gate=rows_per_gate)
            if gate_map is None:
                gate_map = row_map
            if gate_map is not None:
                _require_shape(gate_map, "gate_map", (rows,), torch.int32, dev)
            elif gate_rows * rows_per_gate < rows:
                raise ValueError(f"gate has {gate_rows} rows of {rows_per_gate} rows each, {rows} rows to gate")
    # what other rows, or later ones, read
    read = dict(pre_gamma=pre_gamma, pre_beta=pre_beta, post_gamma=post_gamma, post_beta=post_beta, gate=gate,
                row_map=row_map, gate_map=gate_map, row_count=row_count)
    if routing is not None:
        read.update(weights=routing.weights, routing=routing.plan)
    if sum_out is None:
        sum_out = torch.empty(rows, D, dtype=torch.float32, device=dev)
    else:
        _require_out(sum_out, "sum_out", (rows, D), torch.float32, dev)
        if _overlap(sum_out, x) and (row_map is not None or sum_out.data_ptr() != x.data_ptr()):
            raise ValueError("sum_out may share memory with x only as x itself, without row_map")
        _require_apart(sum_out, "sum_out", branch=branch, **read)
    if out is None:
        out = torch.empty(rows, D, dtype=branch.dtype, device=dev)
    else:
        _require_out(out, "out", (rows, D), branch.dtype, dev)
        if _overlap(out, branch) and (routing is not None or out.data_ptr() != branch.data_ptr()):
            raise ValueError("out may share memory with branch only as branch itself, without routing")
        _require_apart(out, "out", x=x, sum_out=sum_out, **read)
    desc = _lib.SandwichDesc(
        x.data_ptr(), _ptr(row_map), branch.data_ptr(), routing.weights.data_ptr() if routing is not None else None,
        routing.row_slot.data_ptr() if routing is not None else None, _ptr(post_gamma), _ptr(post_beta),
        _ptr(gate), _ptr(gate_map), _ptr(pre_gamma), _ptr(pre_beta), _ptr(row_count), sum_out.data_ptr(),
        out.data_ptr(), branch.shape[0], code, rows, x.shape[0], D, routing.top_k if routing is not None else 0,
        gate_rows, rows_per_gate, gate_code, _GATES[gate_act], 1 if kind == "rms" else 0, eps, residual_scale,
    )
    rc = _launch(dev, _lib.load().tj_sandwich_norm, ctypes.byref(desc))
    _lib.check(rc, "sandwich_norm")
    return sum_out, out
