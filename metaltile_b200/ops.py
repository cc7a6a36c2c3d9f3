"""Typed ops on tensors that already live on the GPU.

PyTorch is used only as the owner of device memory and streams: every function hands raw device pointers and the
current CUDA stream to ``libmtcuda.so``.  The argument checks, the output allocation and the call itself are in the
native binding (``csrc/binding.cpp``): through ctypes they cost 12-18 us a call, more than most decode kernels.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import BF16, F16, F32
from .context import Context

_lib.load()                                  # checks that the library exports what the header declares
try:
    from . import _native
except ImportError as e:
    raise ImportError(f"the native binding of the typed ops is missing ({e}): build it with `python -m metaltile_b200.build` "
                      "(there is no CPU or PyTorch fallback for these ops)") from e

if _native.torch_version != torch.__version__:
    raise ImportError(f"the native binding of the typed ops was compiled against PyTorch {_native.torch_version}, this is {torch.__version__}: "
                      "build it again with `python -m metaltile_b200.build`")

_TORCH_DT = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}

_ctx_cache = {}


def context(device=None) -> Context:
    """The process-wide Context of a device (created on first use)."""
    idx = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    if idx not in _ctx_cache:
        _ctx_cache[idx] = Context(idx)
    return _ctx_cache[idx]


_native.set_context(context)


def _check_dense(w, scales, biases, x, bits, group_size):
    if not (w.is_cuda and scales.is_cuda and biases.is_cuda and x.is_cuda):
        raise ValueError("all operands must be CUDA tensors")
    if w.dtype not in (torch.int32, torch.uint32):
        raise TypeError("w must hold packed 32-bit words (torch.int32 / torch.uint32)")
    if x.dtype not in _TORCH_DT or scales.dtype != x.dtype or biases.dtype != x.dtype:
        raise TypeError("x, scales and biases must share one dtype in {f32, f16, bf16}")
    x2 = x.reshape(-1, x.shape[-1])
    M, K = x2.shape
    N = w.shape[0]
    if w.shape[1] * 32 != K * bits:
        raise ValueError(f"w has {w.shape[1]} words per row, expected K*bits/32 = {K * bits / 32}")
    if scales.shape != (N, K // group_size) or biases.shape != scales.shape:
        raise ValueError("scales/biases must be [N, K/group_size]")
    for t in (w, scales, biases, x2):
        if not t.is_contiguous():
            raise ValueError("operands must be contiguous")
    return x2, M, N, K


def _check_out(out, M, N, like):
    """A caller-supplied output must be the dense row-major [M, N] block the kernels write."""
    if out.device != like.device or out.dtype != like.dtype:
        raise TypeError("out must live on the same device and have the dtype of x")
    if out.numel() != M * N or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous block of M*N = {M * N} elements "
                         "(a column slice of a wider tensor with M > 1 is not)")


def qmv(w, scales, biases, x, bits: int, group_size: int, out=None, ctx: Context = None):
    """out[M, N] = x[M, K] @ dequant(w)[N, K]^T (decode, M <= 16 tuned); ``Context.launch_of`` names the kernel."""
    return _native.dense(0, w, scales, biases, x, bits, group_size, out, ctx)


def qmm(w, scales, biases, x, bits: int, group_size: int, out=None, ctx: Context = None):
    """Like ``qmv`` but routed by M as the reference's ``mt_qmm_for`` does (prefill -> tensor cores)."""
    return _native.dense(1, w, scales, biases, x, bits, group_size, out, ctx)


def _projection(w, scales, biases, x, bits, group_size, outs, phase=0):
    x2, M, N, K = _check_dense(w, scales, biases, x, bits, group_size)
    for o in outs:
        _check_out(o, M, N, x)
    return {"w": w.data_ptr(), "scales": scales.data_ptr(), "biases": biases.data_ptr(), "x": x2.data_ptr(),
            "outs": [o.data_ptr() for o in outs], "M": M, "N": N, "K": K, "bits": bits, "group_size": group_size,
            "dtype": _TORCH_DT[x.dtype], "phase": phase}


def qmv_batched(mats, x, bits: int, group_size: int, out=None, ctx: Context = None):
    """Several projections of the same activations in one launch: ``mats`` = [(w, scales, biases), ...] (1 to 4).

    Returns ``out[M, sum(N_i)]`` with the results side by side - for M = 1 the concatenated vector of
    ``ffai_batched_qkv_qgemv`` (crates/metaltile-std/src/ffai/batched_qkv_qgemv.rs:1-35).  For M > 1 every
    projection writes its own contiguous [M, N_i] tile and the tiles are returned as a list instead.  The f32 sums of a fused
    projection may be added in another order than ``qmv`` of it alone adds them (the last bit of an output may differ); the
    same call always gives the same bits."""
    return _native.qmv_batched(mats, x, bits, group_size, out, ctx)


def unpack_codes(w, K: int, bits: int, ctx: Context = None):
    """u8[N, K] integer codes of a packed matrix (for bit-exact checks)."""
    return _native.unpack_codes(w, K, bits, ctx)


# ---- MoE -----------------------------------------------------------------------------------------
def moe_router_topk(logits, k: int, norm_topk_prob: int = 1, ctx: Context = None):
    """(indices int32[rows, k], weights T[rows, k]) of ``mt_moe_router_topk``."""
    return _native.moe_router_topk(logits, k, norm_topk_prob, ctx)


def moe_sort(topk_idx, n_experts: int, ctx: Context = None):
    """Stable expert sort: (sort_token_idx[T*k], inv_perm[T, k], expert_offsets[E+1], row_expert[T*k]), int32."""
    return _native.moe_sort(topk_idx, n_experts, ctx)


def moe_permute(tokens, sort_token_idx, out=None, ctx: Context = None):
    return _native.moe_permute(tokens, sort_token_idx, out, ctx)


def moe_unpermute(expert_outputs, inv_perm, weights, out=None, ctx: Context = None):
    return _native.moe_unpermute(expert_outputs, inv_perm, weights, out, ctx)


def swiglu(gate, up, out=None, ctx: Context = None):
    return _native.swiglu(gate, up, out, ctx)


def gather_qmm(x, w, scales, biases, bits: int, group_size: int, expert_offsets=None, indices=None, out=None,
               ctx: Context = None):
    """out[t, n] = sum_k x[t, k] * dequant(w[E(t)])[n, k]; x rows sorted by expert; w [E, n_out, k*bits/32]."""
    return _native.gather_qmm(x, w, scales, biases, bits, group_size, expert_offsets, indices, out, ctx)


def moe_experts(x, gate, up, down, bits: int, group_size: int, expert_offsets, sort_token_idx=None, out=None, ctx: Context = None):
    """y[r] = down_e(silu(gate_e(x_r)) * up_e(x_r)) for rows sorted by expert; gate / up / down are (w, scales, biases)
    with w [E, inter, hidden*bits/32] (gate, up) and [E, hidden, inter*bits/32] (down).  ``sort_token_idx`` folds the
    permutation in: row r reads ``x[sort_token_idx[r]]``."""
    return _native.moe_experts(x, gate, up, down, bits, group_size, expert_offsets, sort_token_idx, out, ctx)


def rms_norm_qmv(w, scales, biases, x, norm_weight, eps: float, bits: int, group_size: int, out=None, ctx: Context = None):
    """``qmv(rms_norm(x) * norm_weight)`` in one launch (``ffai_rms_norm_qgemv``,
    crates/metaltile-std/src/ffai/rms_norm_qgemv.rs:51-107): x and norm_weight are vectors of length K, out [1, N]."""
    return _native.rms_norm_qmv(w, scales, biases, x, norm_weight, eps, bits, group_size, out, ctx)


def affine_quantize(w, bits: int, group_size: int, ctx: Context = None):
    """Float tensor ``w [..., K]`` (K a multiple of the group size) -> (packed int32 ``[..., K*bits/32]``, scales, biases
    ``[..., K/group_size]``) in the layout the quantized matmuls read (``mt_affine_quantize_int*``,
    crates/metaltile-std/src/mlx/quantized.rs:3629-3667).  A product of them may follow on the same stream at once: the
    context keeps it from requesting its weights before they are written (other writers: option ``pdl_early_weights``)."""
    return _native.affine_quantize(w, bits, group_size, ctx)


def affine_dequantize(w, scales, biases, bits: int, group_size: int, ctx: Context = None):
    """The inverse of ``affine_quantize``: ``scale * q + bias`` in the type of ``scales`` (``mt_affine_dequantize_int*``)."""
    return _native.affine_dequantize(w, scales, biases, bits, group_size, ctx)


def dequant_gather(weight, scales, biases, indices, bits: int, group_size: int, ctx: Context = None):
    """Rows ``indices`` (int32) of a quantized table ``weight [vocab, hidden*bits/32]`` dequantized: ``[n_tokens, hidden]``
    in the type of ``scales`` (``dequant_gather_int*``, crates/metaltile-std/src/ffai/dequant_gather.rs:44-101)."""
    return _native.dequant_gather(weight, scales, biases, indices, bits, group_size, ctx)


def qvm(w, scales, biases, x, bits: int, group_size: int, out=None, ctx: Context = None):
    """``x @ W`` with W stored transposed and quantized along K: w [K, N*bits/32], scales / biases [K/group_size, N],
    x [M, K] -> out [M, N] (``mt_qvm_*``, crates/metaltile-std/src/mlx/quantized.rs:4397-4530).  Like the other dense products
    it requests its first weights while the previous kernel of the stream drains (option ``pdl_early_weights``)."""
    return _native.qvm(w, scales, biases, x, bits, group_size, out, ctx)


# ---- 8-bit floating point: e4m3 codes with a float32 scale for each block of 128 values ---------------------------------------
def _out_dtype(dtype):
    if dtype is None:
        return -1
    if dtype not in _TORCH_DT:
        raise TypeError("out_dtype must be float32, float16 or bfloat16")
    return _TORCH_DT[dtype]


def fp8_quantize(x, block_rows: int = 1, pow2: bool = False, rows=None, ctx: Context = None):
    """Float tensor -> (codes ``float8_e4m3fn`` like ``x``, scales float32) in the layout the products below read.

    ``block_rows=1``, activations: ``x [.., K]``, one scale for 128 values of a row, ``[.., ceil(K/128)]``; ``rows`` (int32) folds
    ``moe_permute`` in: row r of the result is ``x[rows[r]]``.  ``block_rows=128``, weights: ``x [.., N, K]``, one scale for 128 x 128 values,
    ``[.., ceil(N/128), ceil(K/128)]``.  A scale is ``max(max|x| / 448, 2**-90)`` over the finite values of its block, with ``pow2`` the least power
    of two that is not below that; a code is the e4m3 value nearest to ``x / scale``, ties to even.  Infinities and NaN become NaN."""
    return _native.fp8_quantize(x, block_rows, pow2, rows, ctx)


def fp8_mm(x, w, w_scales, x_scales=None, out_dtype=None, out=None, ctx: Context = None):
    """out[M, N] = x @ w^T with w ``[N, K]`` codes and ``w_scales [ceil(N/128), ceil(K/128)]``, block sums scaled and added in f32.

    ``x [.., K]`` is codes with ``x_scales [.., ceil(K/128)]``, or f32 / f16 / bf16 activations, which are quantized in the call as
    ``fp8_quantize(x)`` does (same result).  ``out_dtype`` (f32, f16, bf16) defaults to the type of float activations, bf16 for codes.
    The gradient of x is the same product with the matrix the other way round, ``fp8_mm(dy, wt, wt_scales)`` with ``wt = w.T.contiguous()`` and
    ``wt_scales = w_scales.T.contiguous()`` - blocks of 128 x 128 stay what they are.  Like the other dense products it requests its first weights
    while the previous kernel of the stream drains (option ``pdl_early_weights``): keep such matrices, or synchronise after making them."""
    return _native.fp8_mm(x, w, w_scales, x_scales, _out_dtype(out_dtype), out, ctx)


def fp8_gather_mm(x, w, w_scales, expert_offsets, x_scales, out_dtype=None, out=None, ctx: Context = None):
    """The grouped form: ``x [rows, K]`` codes sorted by expert (``fp8_quantize(tokens, rows=sort_token_idx)``), w ``[E, N, K]``, w_scales
    ``[E, ceil(N/128), ceil(K/128)]``, ``expert_offsets`` int32 ``[E + 1]`` from ``moe_sort``; out ``[rows, N]``, bf16 by default.  Rows that
    no expert owns keep what ``out`` holds there (anything, where the call makes ``out``)."""
    return _native.fp8_gather_mm(x, w, w_scales, expert_offsets, x_scales, _out_dtype(out_dtype), out, ctx)


# ---- the training side of the router ---------------------------------------------------------------------------------------
def moe_balance(logits, topk_idx, coef: float = 1.0, mask=None, ctx: Context = None):
    """The balance loss of a router over the rows that ``mask`` (bool ``[rows]``) keeps: (loss float32 ``[]``, counts int32 ``[E]``, mean_probs
    float32 ``[E]``, n_counted int32 ``[]``).

    With p = softmax(logits), n rows kept and c_e slots of ``topk_idx [rows, k]`` that name expert e:
    ``loss = coef * E * sum_e c_e / (n k) * mean_t p_te``.  Uniform routing gives ``coef``; no rows give 0."""
    return _native.moe_balance(logits, topk_idx, coef, mask, ctx)


def moe_balance_grad(logits, counts, n_counted, k: int, grad_loss=None, coef: float = 1.0, mask=None, out=None, ctx: Context = None):
    """The gradient of the logits, ``[rows, E]`` in their type, from what ``moe_balance`` returned: ``grad_loss * coef * E / n * p_te *
    (f_e - sum_j f_j p_tj)`` with ``f = counts / (n k)`` constant; zeros for masked rows.  ``grad_loss``: one float32 on the device (None: 1).
    Where several ranks share a batch, add up their ``counts`` and ``n_counted`` first: the gradient is then that of the common loss."""
    return _native.moe_balance_grad(logits, counts, n_counted, k, grad_loss, coef, mask, out, ctx)
