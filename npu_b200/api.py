"""Torch-facing native API over the C ABI: causal GQA prefill, split-KV decode
and the fused RoPE + KV-cache append that feeds them.

These are the B200 entry points behind the reference-compatible wrapper in
npu_b200.fa (NpuAttention.run_batch), and the operators that serve sequences
of different lengths together: attention over packed prompts, a paged KV cache
(append, single-token attention, reading back; bf16 or 8-bit), penalties on
logits and token sampling. Tensors are CUDA bf16 with a contiguous
head dimension, except for prefill_host, which takes host bf16 tensors and
moves them itself; nothing here falls back to a CPU path.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib


def _stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _need_cuda_bf16(name: str, t: torch.Tensor, ndim: int) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (no CPU path exists)")
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} needs a contiguous last (head_dim) dimension")


def _check_gate(gate: torch.Tensor, shape: tuple, device: torch.device) -> None:
    if not isinstance(gate, torch.Tensor) or gate.device != device:
        raise ValueError("gate must be a CUDA tensor on q's device")
    if gate.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("gate must be float32 or bfloat16")
    if tuple(gate.shape) != tuple(shape) or gate.stride(-1) != 1:
        raise ValueError(f"gate must be {list(shape)} with a contiguous last dim, got {tuple(gate.shape)}")


def prefill(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    start_pos: int = 0,
    start_pos_per_batch: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    causal: bool = True,
    out_dtype: torch.dtype = torch.float32,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    gate: Optional[torch.Tensor] = None,
):
    """Attention forward for q [B, Hq, Tq, D] against k/v [B, Hkv, Tk, D].

    Row r of q sits at absolute position start + r (start = start_pos, or
    start_pos_per_batch[b] if given as an int32 CUDA tensor [B]). With causal,
    key c is masked iff c > start + r; rows with no key output 0 — the
    semantics of flash_attention_ref (npu/fa_ref.py:42-131). Query head h uses
    KV head h // (Hq // Hkv). Returns o [B, Hq, Tq, D] in out_dtype (and the
    natural-log LSE [B, Hq, Tq] if return_lse). With `gate` ([B, Hq, Tq, D],
    fp32 or bf16, any strides with a contiguous last dim) the output is
    attention * sigmoid(gate), fused into the kernel's stores (Qwen's gated
    attention, qwen/forward.py:223-226).
    """
    _need_cuda_bf16("q", q, 4)
    _need_cuda_bf16("k", k, 4)
    _need_cuda_bf16("v", v, 4)
    B, Hq, Tq, D = q.shape
    Bk, Hkv, Tk, Dk = k.shape
    if (Bk, Dk) != (B, D) or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("out_dtype must be float32 or bfloat16")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, Hq, Tq, D), dtype=out_dtype, device=q.device)
    elif out.dtype != out_dtype or tuple(out.shape) != (B, Hq, Tq, D) or out.stride(-1) != 1:
        raise ValueError("out must match [B, Hq, Tq, D], out_dtype and a contiguous last dim")
    lse = torch.empty((B, Hq, Tq), dtype=torch.float32, device=q.device) if return_lse else None
    spb = None
    if start_pos_per_batch is not None:
        spb = start_pos_per_batch
        if spb.dtype != torch.int32 or spb.device != q.device or spb.numel() != B or not spb.is_contiguous():
            raise ValueError("start_pos_per_batch must be a contiguous int32 tensor [B] on q's device")
    lib = _lib.load()
    if gate is not None:
        _check_gate(gate, (B, Hq, Tq, D), q.device)
    with torch.cuda.device(q.device):
        if gate is None:
            rc = lib.b2a_prefill(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                lse.data_ptr() if lse is not None else None,
                B, Hq, Hkv, Tq, Tk, D,
                _lib.ll3(*q.stride()[:3]), _lib.ll3(*k.stride()[:3]), _lib.ll3(*v.stride()[:3]),
                _lib.ll3(*out.stride()[:3]),
                int(start_pos), spb.data_ptr() if spb is not None else None,
                float(scale), 1 if causal else 0, 1 if out_dtype == torch.float32 else 0,
                _stream_ptr(q.device),
            )
        else:
            rc = lib.b2a_prefill_gated(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), gate.data_ptr(), out.data_ptr(),
                lse.data_ptr() if lse is not None else None,
                B, Hq, Hkv, Tq, Tk, D,
                _lib.ll3(*q.stride()[:3]), _lib.ll3(*k.stride()[:3]), _lib.ll3(*v.stride()[:3]),
                _lib.ll3(*gate.stride()[:3]), _lib.ll3(*out.stride()[:3]),
                1 if gate.dtype == torch.bfloat16 else 0,
                int(start_pos), spb.data_ptr() if spb is not None else None,
                float(scale), 1 if causal else 0, 1 if out_dtype == torch.float32 else 0,
                _stream_ptr(q.device),
            )
    _lib.check(rc, "b2a_prefill")
    return (out, lse) if return_lse else out


def prefill_host_workspace_bytes(B: int, Hq: int, Hkv: int, Tq: int, Tk: int, D: int,
                                 out_fp32: bool = False, n_chunks: int = 0) -> int:
    return int(_lib.load().b2a_prefill_host_workspace_bytes(B, Hq, Hkv, Tq, Tk, D, 1 if out_fp32 else 0,
                                                            n_chunks))


def prefill_host(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    start_pos: int = 0,
    start_pos_per_batch=None,
    scale: Optional[float] = None,
    causal: bool = True,
    out_dtype: torch.dtype = torch.bfloat16,
    out: Optional[torch.Tensor] = None,
    n_chunks: int = 0,
    device: Optional[torch.device] = None,
    workspace: Optional[torch.Tensor] = None,
    sync: bool = True,
) -> torch.Tensor:
    """`prefill` for tensors in HOST memory (b2a_prefill_host): q [B, Hq, Tq, D]
    and k/v [B, Hkv, Tk, D] contiguous bf16 CPU tensors, result o [B, Hq, Tq, D]
    on the host (page-locked when allocated here). The work is cut into
    n_chunks pieces whose uploads, kernels and downloads overlap on the GPU
    `device` (default: the current one). start_pos_per_batch, if given, is a
    host sequence / CPU int32 tensor [B]. With sync=False the call returns once
    the copies and kernels are queued on the device's current stream; the
    inputs must then stay untouched and `out` unread until that stream is
    synchronised. Page-locked inputs (`tensor.pin_memory()`) are needed for the
    copies to overlap; pageable ones give the same result, serialised.
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.is_cuda:
            raise ValueError(f"{name} must be a CPU tensor (use prefill for device tensors)")
        if t.dtype != torch.bfloat16 or t.dim() != 4 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous 4-d bfloat16 tensor, got {t.dtype} {tuple(t.shape)}")
    B, Hq, Tq, D = q.shape
    Bk, Hkv, Tk, Dk = k.shape
    if (Bk, Dk) != (B, D) or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("out_dtype must be float32 or bfloat16")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is not None and (out.is_cuda or out.dtype != out_dtype or tuple(out.shape) != (B, Hq, Tq, D)
                            or not out.is_contiguous()):
        raise ValueError("out must be a contiguous CPU tensor [B, Hq, Tq, D] of out_dtype")
    spb = None
    if start_pos_per_batch is not None:
        if isinstance(start_pos_per_batch, torch.Tensor) and start_pos_per_batch.is_cuda:
            raise ValueError("start_pos_per_batch must be on the host")
        spb = torch.as_tensor(start_pos_per_batch, dtype=torch.int32).contiguous()
        if spb.numel() != B:
            raise ValueError("start_pos_per_batch must be a host sequence of B int32 positions")
    if device is None:
        if not torch.cuda.is_available():
            raise RuntimeError("prefill_host needs a CUDA device (no CPU path)")
        device = torch.device("cuda", torch.cuda.current_device())
    device = torch.device(device)
    if out is None:
        out = torch.empty((B, Hq, Tq, D), dtype=out_dtype, pin_memory=True)
    out_fp32 = out_dtype == torch.float32
    lib = _lib.load()
    need = int(lib.b2a_prefill_host_workspace_bytes(B, Hq, Hkv, Tq, Tk, D, 1 if out_fp32 else 0, n_chunks))
    if need == 0:
        _lib.check(_lib.B2A_ERR_INVALID_ARG, "b2a_prefill_host_workspace_bytes")
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif not workspace.is_cuda or workspace.device != device or workspace.numel() < need:
        raise ValueError(f"workspace must be a CUDA uint8 tensor of >= {need} bytes on {device}")
    with torch.cuda.device(device):
        rc = lib.b2a_prefill_host(
            q.data_ptr(), k.data_ptr() if Tk else None, v.data_ptr() if Tk else None, out.data_ptr(),
            B, Hq, Hkv, Tq, Tk, D, int(start_pos), spb.data_ptr() if spb is not None else None,
            float(scale), 1 if causal else 0, 1 if out_fp32 else 0, int(n_chunks),
            workspace.data_ptr(), workspace.numel(), _stream_ptr(device),
        )
        _lib.check(rc, "b2a_prefill_host")
        if sync:
            torch.cuda.current_stream(device).synchronize()
    return out


def decode_workspace_bytes(B: int, Hq: int, Hkv: int, D: int, Lmax: int, split_len: int = 0) -> int:
    return int(_lib.load().b2a_decode_workspace_bytes(B, Hq, Hkv, D, Lmax, split_len))


def decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seqlens: torch.Tensor,
    *,
    scale: Optional[float] = None,
    out_dtype: torch.dtype = torch.float32,
    split_len: int = 0,
    workspace: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One query token per sequence: q [B, Hq, D] against caches [B, Hkv, Lmax, D].

    Sequence b attends to keys 0 .. seqlens[b]-1 with no mask (the T=1 path of
    smollm.py:222-234). seqlens is an int32 CUDA tensor [B]. The split-KV
    scratch is taken from `workspace` (a uint8 CUDA tensor) or allocated here
    through torch's caching allocator. With `gate` ([B, Hq, D], fp32 or bf16)
    the output is attention * sigmoid(gate), fused into the combine kernel.
    """
    _need_cuda_bf16("q", q, 3)
    _need_cuda_bf16("k_cache", k_cache, 4)
    _need_cuda_bf16("v_cache", v_cache, 4)
    B, Hq, D = q.shape
    Bk, Hkv, Lmax, Dk = k_cache.shape
    if (Bk, Dk) != (B, D) or tuple(v_cache.shape) != tuple(k_cache.shape):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k_cache.shape)} v{tuple(v_cache.shape)}")
    if seqlens.dtype != torch.int32 or seqlens.device != q.device or seqlens.numel() != B:
        raise ValueError("seqlens must be an int32 tensor [B] on q's device")
    seqlens = seqlens.contiguous()
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    lib = _lib.load()
    if split_len == 0:
        split_len = int(lib.b2a_decode_default_split(B, Hkv, Lmax))
    need = int(lib.b2a_decode_workspace_bytes(B, Hq, Hkv, D, Lmax, split_len))
    if need == 0:
        raise _lib.B2AError(_lib.B2A_ERR_INVALID_ARG, "b2a_decode_workspace_bytes")
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=out_dtype, device=q.device)
    if gate is not None:
        _check_gate(gate, (B, Hq, D), q.device)
    with torch.cuda.device(q.device):
        if gate is None:
            rc = lib.b2a_decode(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), seqlens.data_ptr(), out.data_ptr(),
                B, Hq, Hkv, Lmax, D,
                _lib.ll2(*q.stride()[:2]), _lib.ll3(*k_cache.stride()[:3]), _lib.ll3(*v_cache.stride()[:3]),
                _lib.ll2(*out.stride()[:2]),
                float(scale), int(split_len), 1 if out.dtype == torch.float32 else 0,
                workspace.data_ptr(), need, _stream_ptr(q.device),
            )
        else:
            rc = lib.b2a_decode_gated(
                q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), seqlens.data_ptr(), gate.data_ptr(),
                out.data_ptr(), B, Hq, Hkv, Lmax, D,
                _lib.ll2(*q.stride()[:2]), _lib.ll3(*k_cache.stride()[:3]), _lib.ll3(*v_cache.stride()[:3]),
                _lib.ll2(*gate.stride()[:2]), _lib.ll2(*out.stride()[:2]),
                1 if gate.dtype == torch.bfloat16 else 0,
                float(scale), int(split_len), 1 if out.dtype == torch.float32 else 0,
                workspace.data_ptr(), need, _stream_ptr(q.device),
            )
    _lib.check(rc, "b2a_decode")
    return out


def decode_proj(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seqlens: torch.Tensor,
    wo: torch.Tensor,
    x: torch.Tensor,
    *,
    scale: Optional[float] = None,
    split_len: int = 0,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Decode attention fused with the output projection and residual add
    (b2a_decode_proj): x += attention(q, caches) @ wo.T, in place.

    q [B, Hq, D] and the caches as `decode`; wo [dim, Hq * D] (the F.linear
    weight of the output projection, fp32 or bf16, last dim contiguous); x the
    residual stream [B, dim] (fp32 or bf16, last dim contiguous), returned.
    The attention output is rounded to x's dtype before the projection, as
    the unfused `x + F.linear(o, wo)` would see it; every output has one
    writer and a fixed summation order (reproducible results).
    """
    _need_cuda_bf16("q", q, 3)
    _need_cuda_bf16("k_cache", k_cache, 4)
    _need_cuda_bf16("v_cache", v_cache, 4)
    B, Hq, D = q.shape
    Bk, Hkv, Lmax, Dk = k_cache.shape
    if (Bk, Dk) != (B, D) or tuple(v_cache.shape) != tuple(k_cache.shape):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k_cache.shape)} v{tuple(v_cache.shape)}")
    if seqlens.dtype != torch.int32 or seqlens.device != q.device or seqlens.numel() != B:
        raise ValueError("seqlens must be an int32 tensor [B] on q's device")
    for name, t in (("wo", wo), ("x", x)):
        if not isinstance(t, torch.Tensor) or t.device != q.device or t.dim() != 2 or t.stride(-1) != 1:
            raise ValueError(f"{name} must be a 2-d CUDA tensor on q's device with a contiguous last dim")
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"{name} must be float32 or bfloat16")
    dim = wo.shape[0]
    if wo.shape[1] != Hq * D or tuple(x.shape) != (B, dim):
        raise ValueError(f"wo must be [dim, {Hq * D}] and x [{B}, dim], got wo{tuple(wo.shape)} x{tuple(x.shape)}")
    seqlens = seqlens.contiguous()
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    lib = _lib.load()
    if split_len == 0:
        split_len = int(lib.b2a_decode_default_split(B, Hkv, Lmax))
    need = int(lib.b2a_decode_workspace_bytes(B, Hq, Hkv, D, Lmax, split_len))
    if need == 0:
        raise _lib.B2AError(_lib.B2A_ERR_INVALID_ARG, "b2a_decode_workspace_bytes")
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        rc = lib.b2a_decode_proj(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), seqlens.data_ptr(), wo.data_ptr(),
            wo.stride(0), 1 if wo.dtype == torch.float32 else 0, dim, x.data_ptr(), x.stride(0),
            1 if x.dtype == torch.float32 else 0, B, Hq, Hkv, Lmax, D,
            _lib.ll2(*q.stride()[:2]), _lib.ll3(*k_cache.stride()[:3]), _lib.ll3(*v_cache.stride()[:3]),
            float(scale), int(split_len), workspace.data_ptr(), need, _stream_ptr(q.device),
        )
    _lib.check(rc, "b2a_decode_proj")
    return x


def rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    start_pos: int = 0,
    start_pos_per_batch: Optional[torch.Tensor] = None,
    seqlens_out: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
    q_norm: Optional[torch.Tensor] = None,
    k_norm: Optional[torch.Tensor] = None,
    norm_eps: float = 1e-6,
    rope_dim: Optional[int] = None,
) -> torch.Tensor:
    """Rotate q and k and append k, v to a device-resident cache, in place.

    q [B, T, Hq, D], k and v [B, T, Hkv, D] (fp32 or bf16, last dim
    contiguous; typically views of one fused QKV projection) are rotated with
    the rotary tables cos/sin [max_pos, D] (same dtype, rotate-half form of
    smollm.py:53-58) at positions p_b + t, p_b = start_pos_per_batch[b] or
    start_pos. k and v land in rows p_b .. p_b + T - 1 of k_cache/v_cache
    [B, Hkv, Lmax, D] bf16; seqlens_out (int32 [B], optional) receives
    p_b + T. Returns q rotated as [B, Hq, T, D] bf16, the layout prefill and
    decode take.

    Qwen's gated-attention prologue (qwen/forward.py:178-204): q_norm /
    k_norm ([D], q's dtype) RMS-normalise each q / k head first (eps
    norm_eps), and rope_dim < D rotates only the first rope_dim lanes (cos/sin
    are then [max_pos, rope_dim]).
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda or t.dim() != 4 or t.stride(-1) != 1:
            raise ValueError(f"{name} must be a CUDA [B, T, H, D] tensor with a contiguous last dim")
    if q.dtype not in (torch.float32, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share one dtype, float32 or bfloat16")
    if cos.dtype != q.dtype or sin.dtype != q.dtype or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("cos/sin must be contiguous [max_pos, D] tensors in q's dtype")
    _need_cuda_bf16("k_cache", k_cache, 4)
    _need_cuda_bf16("v_cache", v_cache, 4)
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    Bc, Hc, Lmax, Dc = k_cache.shape
    if tuple(k.shape) != (B, T, Hkv, D) or tuple(v.shape) != (B, T, Hkv, D):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if (Bc, Hc, Dc) != (B, Hkv, D) or tuple(v_cache.shape) != tuple(k_cache.shape):
        raise ValueError(f"cache shape {tuple(k_cache.shape)} does not fit k{tuple(k.shape)}")
    rope_dim = D if rope_dim is None else int(rope_dim)
    if cos.dim() != 2 or cos.shape[1] != rope_dim or tuple(sin.shape) != tuple(cos.shape):
        raise ValueError("cos/sin must be [max_pos, rope_dim]")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.dtype != q.dtype or w.device != q.device or tuple(w.shape) != (D,)
                              or not w.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous [D] tensor in q's dtype on q's device")
    spb = None
    if start_pos_per_batch is not None:
        spb = start_pos_per_batch
        if spb.dtype != torch.int32 or spb.device != q.device or spb.numel() != B or not spb.is_contiguous():
            raise ValueError("start_pos_per_batch must be a contiguous int32 tensor [B] on q's device")
    if seqlens_out is not None:
        if (seqlens_out.dtype != torch.int32 or seqlens_out.device != q.device or seqlens_out.numel() != B
                or not seqlens_out.is_contiguous()):
            raise ValueError("seqlens_out must be a contiguous int32 tensor [B] on q's device")
    if q_out is None:
        q_out = torch.empty((B, Hq, T, D), dtype=torch.bfloat16, device=q.device)
    elif q_out.dtype != torch.bfloat16 or tuple(q_out.shape) != (B, Hq, T, D) or not q_out.is_contiguous():
        raise ValueError("q_out must be a contiguous bf16 [B, Hq, T, D] tensor")
    lib = _lib.load()
    with torch.cuda.device(q.device):
        rc = lib.b2a_qk_norm_rope_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(),
            _lib.ll3(*q.stride()[:3]), _lib.ll3(*k.stride()[:3]), _lib.ll3(*v.stride()[:3]),
            1 if q.dtype == torch.bfloat16 else 0,
            q_norm.data_ptr() if q_norm is not None else None,
            k_norm.data_ptr() if k_norm is not None else None, float(norm_eps),
            cos.data_ptr(), sin.data_ptr(), cos.shape[0], rope_dim,
            q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            _lib.ll3(*k_cache.stride()[:3]), _lib.ll3(*v_cache.stride()[:3]),
            B, T, Hq, Hkv, D, Lmax, int(start_pos),
            spb.data_ptr() if spb is not None else None,
            seqlens_out.data_ptr() if seqlens_out is not None else None,
            _stream_ptr(q.device),
        )
    _lib.check(rc, "b2a_qk_norm_rope_append")
    return q_out


def _serving():
    """The compiled binding of the serving operators (loaded with the library, never replaced by a fallback)."""
    global _serving_module
    if _serving_module is None:
        _lib.load()
        try:
            from . import _serving as module
        except ImportError as e:
            raise _lib.B2AError(_lib.B2A_ERR_CUDA,
                                f"_serving is not built (run `python -m npu_b200.build`): {e}") from e
        _serving_module = module
    return _serving_module


_serving_module = None


def prefill_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    *,
    scale: Optional[float] = None,
    causal: bool = True,
    out_dtype: torch.dtype = torch.float32,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    gate: Optional[torch.Tensor] = None,
):
    """`prefill` over sequences of different lengths packed along one axis:
    q [Nq, Hq, D] against k/v [Nk, Hkv, D].

    Sequence b owns query rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 and
    the keys that cu_seqlens_k (default: cu_seqlens_q) gives the same way;
    both are int32 CUDA tensors [B + 1], and the lengths are never read by the
    host. With causal, a sequence's last query sees all its keys (row r sees
    keys up to keys - queries + r); rows that see no key give 0. Rows outside
    every sequence are not written. Returns o [Nq, Hq, D] in out_dtype (and the
    natural-log LSE [Hq, Nq] if return_lse); `gate` ([Nq, Hq, D], fp32 or bf16)
    multiplies the output by sigmoid(gate) as in `prefill`.
    """
    return _serving().prefill_varlen(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal, out_dtype, out, return_lse,
                                     gate)


def decode_paged_workspace_bytes(B: int, Hq: int, Hkv: int, D: int) -> int:
    return int(_lib.load().b2a_decode_paged_workspace_bytes(B, Hq, Hkv, D))


def decode_paged(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seqlens: torch.Tensor,
    *,
    scale: Optional[float] = None,
    out_dtype: torch.dtype = torch.float32,
    workspace: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """`decode` over a paged cache: q [B, Hq, D] against page pools
    [n_pages, Hkv, page, D] (bf16, page a multiple of 16; any stored order with
    a contiguous last dim).

    Key j of sequence b is slot j % page of page block_table[b, j // page]
    (int32 CUDA tensor [B, pages]; entries past the last page of a sequence
    are not read), and keys 0 .. seqlens[b] - 1 are attended; a sequence without
    keys gives 0. Slots past a sequence's end may hold anything. The lengths
    stay on the device; scratch comes from `workspace` (a uint8 CUDA tensor of
    decode_paged_workspace_bytes) or torch's allocator. `gate` ([B, Hq, D])
    as in `decode`. With k_scales and v_scales the pools are 8-bit
    (float8_e4m3fn), as `rope_append_paged` writes them.
    """
    return _serving().decode_paged(q, k_pages, v_pages, block_table, seqlens, scale, out_dtype, workspace, out, gate,
                                   k_scales, v_scales)


def decode_paged_shared_workspace_bytes(B: int, Hq: int, Hkv: int, D: int, n_groups: int = 1) -> int:
    return int(_lib.load().b2a_decode_paged_shared_workspace_bytes(B, Hq, Hkv, D, n_groups))


def decode_paged_shared(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seqlens: torch.Tensor,
    prefix_lens: torch.Tensor,
    cu_groups: Optional[torch.Tensor] = None,
    *,
    scale: Optional[float] = None,
    out_dtype: torch.dtype = torch.float32,
    workspace: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    min_saved_bytes: Optional[int] = None,
) -> torch.Tensor:
    """`decode_paged` for sequences that share the first keys of their cache (a
    system prompt, a document many ask about): the same result, with the shared
    keys read once for a group and attended as one matrix product.

    Group g is the sequences cu_groups[g] .. cu_groups[g + 1] - 1 (int32 CUDA
    tensor [groups + 1]; None: all sequences are one group), whose first
    prefix_lens[g] keys (int32 CUDA tensor [groups]) are the same: block_table
    names them for every sequence, and any of a group's rows may be read. Whole
    blocks of 64 keys are shared; a sequence that is alone in its group, in none,
    or shorter than the prefix attends by itself. Both tensors are read on the
    device. bf16 pools. P is rounded to bf16 over the shared keys, as in
    `prefill`. workspace: decode_paged_shared_workspace_bytes.

    Where sharing would save reading fewer than min_saved_bytes bytes of keys and
    values nothing is shared. The default is 36 MB, and 160 MB if all sequences but
    one of each group shared all that block_table can name (else the call is
    `decode_paged`'s), about where the launches were measured to pay. The host sees
    the table's width only: with tables much wider than the sequences a call that
    has little to share takes 6 to 13 us longer than `decode_paged` (up to 1.75
    times as long), and with small groups a call can be a third slower. A server that
    knows its shapes sets min_saved_bytes (0: share whatever there is) or calls
    `decode_paged`. Whether keys are shared also decides how P is rounded.
    """
    return _serving().decode_paged_shared(q, k_pages, v_pages, block_table, seqlens, prefix_lens, cu_groups, scale,
                                          out_dtype, workspace, out, gate, min_saved_bytes)


def gather_paged(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    n_tokens: int,
    *,
    start_pos: int = 0,
    start_pos_per_batch: Optional[torch.Tensor] = None,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
    v_out: Optional[torch.Tensor] = None,
):
    """Cached keys and values as packed rows (k, v), each [n_tokens, Hkv, D]
    bf16: what `prefill_varlen` reads, for prompts that continue cached ones.

    Row n of sequence b (cu_seqlens[b] <= n < cu_seqlens[b + 1]; int32 CUDA
    tensor [B + 1], read on the device) is the key at position p_b + n -
    cu_seqlens[b], p_b = start_pos_per_batch[b] or start_pos; pools, scales and
    block_table as `decode_paged`. 8-bit values are multiplied by their scale in
    fp32 and rounded once. Rows outside every sequence are not written (those of
    tensors made here hold anything); a position without a page gives zeros and
    shows in `device_error()`.
    """
    return _serving().gather_paged(k_pages, v_pages, block_table, cu_seqlens, n_tokens, start_pos,
                                   start_pos_per_batch, k_scales, v_scales, k_out, v_out)


def rope_append_paged(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    start_pos: int = 0,
    start_pos_per_batch: Optional[torch.Tensor] = None,
    seqlens_out: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
    q_norm: Optional[torch.Tensor] = None,
    k_norm: Optional[torch.Tensor] = None,
    norm_eps: float = 1e-6,
    rope_dim: Optional[int] = None,
    return_kv: bool = False,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
):
    """`rope_append` for packed tokens and a paged cache: q [N, Hq, D], k and v
    [N, Hkv, D] (fp32 or bf16, last dim contiguous; typically views of one fused
    QKV projection), pools and block_table as `decode_paged`.

    Token n of sequence b (cu_seqlens[b] <= n < cu_seqlens[b + 1]) is at
    position p_b + n - cu_seqlens[b], p_b = start_pos_per_batch[b] or
    start_pos; its k and v go to the page and slot of that position, which
    block_table must already name. seqlens_out (int32 [B], optional, not the
    tensor start_pos_per_batch, which is read while it is written) receives
    p_b + tokens. cos/sin [max_pos, rope_dim] are fp32 or q's dtype; the
    arithmetic is fp32 and rounds to bf16 once. q_norm, k_norm, norm_eps and
    rope_dim as in `rope_append`. Returns q rotated, [N, Hq, D] bf16; with
    return_kv (q, k, v): k rotated and v as packed bf16 [N, Hkv, D] for
    `prefill_varlen` (v itself when it is bf16 already).

    With k_scales and v_scales ([n_pages, Hkv, page] fp32, contiguous slots) the
    pools are 8-bit (float8_e4m3fn): each token's k and v of a KV head, a row y
    of D values, is stored as e4m3(y * (1 / s)) with s = max(max |y| / 448, 2^-100)
    beside it, both quotients rounded to fp32, from the fp32 values. A row with an infinity or a NaN reads back as NaN.
    """
    return _serving().rope_append_paged(q, k, v, cos, sin, k_pages, v_pages, block_table, cu_seqlens, start_pos,
                                        start_pos_per_batch, seqlens_out, q_out, q_norm, k_norm, norm_eps, rope_dim,
                                        return_kv, k_scales, v_scales)


def penalize(
    logits: torch.Tensor,
    tokens: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
    *,
    prompt_lengths: Optional[torch.Tensor] = None,
    repetition=1.0,
    frequency=0.0,
    presence=0.0,
    bias: Optional[torch.Tensor] = None,
    allowed: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Penalties for repeated tokens, a bias and a mask on logits [R, V] (fp32 or
    bf16), before `sample`.

    Row r has the tokens tokens[r, : lengths[r]] (int32 or int64 CUDA tensor
    [R, L], any strides; lengths: int32 CUDA tensor [R], default all L), of which
    the first prompt_lengths[r] (default none) are its prompt. Ids outside the
    vocabulary count for nothing. For token v, found c times after the prompt:

      y = x / repetition if x > 0 else x * repetition    if v is among all of them
      y = y - frequency * c - (presence if c > 0 else 0)
      y = y + bias[v]                  bias [V] or [R, V] fp32
      y = -inf                         unless bit v % 32 of allowed[v // 32] is set

    allowed is an int32 tensor [ceil(V / 32)] or [R, ceil(V / 32)] of 32 tokens a
    word. repetition (above 0), frequency and presence are numbers or per-row fp32
    CUDA tensors. Each step is rounded in fp32, the result to the logits' type.
    `out` may be the logits themselves and overlaps no other input. A row whose mask leaves nothing is -inf
    throughout, and `sample` gives -1 for it.
    """
    return _serving().penalize(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed,
                               out)


def sample(
    logits: torch.Tensor,
    noise: Optional[torch.Tensor] = None,
    *,
    temperature=1.0,
    top_k=0,
    top_p=1.0,
    min_p=0.0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The next token of each row of logits [R, V] (fp32 or bf16), int64 [R].

    noise [R, V] fp32 holds independent Exp(1) draws, all above 0
    (`torch.empty(R, V).exponential_()`); the same noise gives the same tokens.
    A row's temperature T, top_k, top_p and min_p are numbers or per-row CUDA
    tensors (fp32; top_k int32). With w = exp((x - max) / T), tokens ranked by
    logit (lowest index first among equals): token j is kept iff fewer than
    top_k tokens rank ahead of it (0: no limit), the weight ahead of it is
    below top_p of the total (1: no limit) and w_j >= min_p; the first always.
    Each filter is taken of the whole distribution. The result is
    argmax w / noise over the kept tokens, so token i comes up with probability
    w_i / (sum of the kept w). T <= 0 (or no noise) gives the argmax. NaN logits
    count as -inf; a row without a logit above -inf gives -1.
    """
    return _serving().sample(logits, noise, temperature, top_k, top_p, min_p, out)


def device_error(clear: bool = True, device: Optional[torch.device] = None) -> int:
    """Status the kernels left in the device error word (synchronises)."""
    import ctypes

    device = device or torch.device("cuda", torch.cuda.current_device())
    st = ctypes.c_int(0)
    with torch.cuda.device(device):
        _lib.check(_lib.load().b2a_get_device_error(ctypes.byref(st), 1 if clear else 0, _stream_ptr(device)),
                   "b2a_get_device_error")
    return st.value
