"""Torch-facing wrappers of the sm_100a task operators.

Each function takes CUDA tensors laid out as the task's OpSpec declares (row-major,
contiguous), allocates the output if none is given, and enqueues the kernel on the current
torch CUDA stream through the C ABI.  There is no fallback: a CPU tensor, a wrong dtype or a
missing native library raises.
"""

from __future__ import annotations

import functools
import operator

import torch

from . import _native

_TORCH_DTYPES = {torch.float16: "fp16", torch.bfloat16: "bf16", torch.float32: "fp32", torch.int32: "i32"}


def dtype_name(t: torch.Tensor) -> str:
    try:
        return _TORCH_DTYPES[t.dtype]
    except KeyError as exc:
        raise TypeError(f"unsupported dtype {t.dtype}") from exc


def _check(t: torch.Tensor, name: str, dtype: torch.dtype | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous (row-major)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _tensor_device(fn):
    """Run an operator on the GPU its tensors live on.

    The C ABI launches on the calling thread's current CUDA device and caches per-device state
    (SM count, kernel attributes) under it, while the stream comes from the tensors' device; so the
    call is made with that device current.  Tensors on two different GPUs are refused (a kernel
    would read the other GPU's memory); CPU tensors are left to each operator's own check, which
    refuses them."""

    @functools.wraps(fn)
    def wrapper(*args, **kwargs):
        devices = {a.device for a in (*args, *kwargs.values()) if isinstance(a, torch.Tensor) and a.is_cuda}
        if len(devices) > 1:
            raise ValueError(f"{fn.__name__}: tensors on more than one device ({', '.join(sorted(map(str, devices)))})")
        if not devices:
            return fn(*args, **kwargs)
        with torch.cuda.device(devices.pop()):
            return fn(*args, **kwargs)

    return wrapper


@_tensor_device
def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y = x * rsqrt(mean(x^2, -1) + eps) * w`` (tasks/rmsnorm/reference.py:110-115)."""
    _check(x, "x")
    _check(w, "w", x.dtype)
    hidden = x.shape[-1] if x.dim() else 1
    if w.numel() != hidden:
        raise ValueError(f"w has {w.numel()} elements, expected hidden={hidden}")
    rows = x.numel() // max(hidden, 1)
    if out is None:
        out = torch.empty_like(x)
    _check(out, "out", x.dtype)
    _native.call(
        "sf_rmsnorm",
        x.data_ptr(),
        w.data_ptr(),
        out.data_ptr(),
        rows,
        hidden,
        float(eps),
        _native.DTYPE_CODES[dtype_name(x)],
        _stream(x),
    )
    return out


@_tensor_device
def gemm_nt(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``C = A @ B^T`` with A ``[M, K]`` and B ``[N, K]`` (fp32 accumulation, one rounding)."""
    _check(a, "A")
    _check(b, "B", a.dtype)
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"gemm_nt needs A [M,K] and B [N,K], got {tuple(a.shape)} and {tuple(b.shape)}")
    m, k = a.shape
    n = b.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _check(out, "out", a.dtype)
    desc = _native.op_desc("gemm_nt", dtype_name(a), dims=(m, n, k), variant=variant)
    _native.run_op(desc, [a.data_ptr(), b.data_ptr(), out.data_ptr()], _stream(a))
    return out


@_tensor_device
def gemm_nn(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
            variant: int = 0) -> torch.Tensor:
    """``C = A @ B`` with A ``[M, K]`` and B ``[K, N]`` (tasks/gemm/reference.py:110-114).

    The tensor-core kernel reads B in place when N % 8 == 0; otherwise ``workspace`` (uint8, at
    least ``gemm_nn_workspace_bytes``, allocated here when not given) receives a transposed copy of
    B first.  Pass ``variant=2`` to force the general kernel."""
    return _gemm_kn("gemm_nn", a, b, out, workspace, variant)


@_tensor_device
def gemm_silu(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
              variant: int = 0) -> torch.Tensor:
    """``C = silu(A @ B)``, silu(v) = v * sigmoid(v) on the fp32 product (tasks/gemm_silu/reference.py,
    ``reference``).  Layouts, workspace and variants as :func:`gemm_nn`; the SiLU is fused into the
    GEMM's epilogue."""
    return _gemm_kn("gemm_silu", a, b, out, workspace, variant)


def _gemm_kn(op: str, a: torch.Tensor, b: torch.Tensor, out, workspace, variant: int) -> torch.Tensor:
    _check(a, "A")
    _check(b, "B", a.dtype)
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError(f"{op} needs A [M,K] and B [K,N], got {tuple(a.shape)} and {tuple(b.shape)}")
    m, k = a.shape
    n = b.shape[1]
    if out is None:
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _check(out, "out", a.dtype)
    need = gemm_nn_workspace_bytes(m, n, k, dtype_name(a))
    if workspace is None and variant != 2 and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=a.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else 0
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    desc = _native.op_desc(op, dtype_name(a), dims=(m, n, k, ws_bytes), variant=variant)
    _native.run_op(desc, [a.data_ptr(), b.data_ptr(), out.data_ptr(), ws_ptr], _stream(a))
    return out


def gemm_nn_workspace_bytes(m: int, n: int, k: int, dtype: str) -> int:
    return int(_native.load().sf_gemm_nn_workspace_bytes(m, n, k, _native.DTYPE_CODES[dtype]))


def kernel_status(device: torch.device | None = None) -> tuple[int, int]:
    """Read and clear the tensor-core kernels' status word of ``device`` (default: the current
    device; synchronises that device's current stream)."""
    if device is None:
        return _native.kernel_status(torch.cuda.current_stream().cuda_stream)
    with torch.cuda.device(device):
        return _native.kernel_status(torch.cuda.current_stream(device).cuda_stream)


def _run(op: str, t: torch.Tensor, ptrs, dims=(), attrs=(), variant: int = 0, flags: int = 0) -> None:
    desc = _native.op_desc(op, dtype_name(t), dims=dims, attrs=attrs, variant=variant, flags=flags)
    _native.run_op(desc, ptrs, _stream(t))


@_tensor_device
def silu(x: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``y = x * sigmoid(x)`` (tasks/silu/reference.py:105-108), any shape, element-wise."""
    _check(x, "x")
    out = torch.empty_like(x) if out is None else out
    _check(out, "out", x.dtype)
    _run("silu", x, [x.data_ptr(), out.data_ptr()], dims=(x.numel(),), variant=variant)
    return out


@_tensor_device
def swiglu(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``y = gate * sigmoid(gate) * up`` (tasks/swiglu/reference.py:109-113)."""
    _check(gate, "gate")
    _check(up, "up", gate.dtype)
    if up.numel() != gate.numel():
        raise ValueError("gate and up must have the same number of elements")
    out = torch.empty_like(gate) if out is None else out
    _check(out, "out", gate.dtype)
    _run("swiglu", gate, [gate.data_ptr(), up.data_ptr(), out.data_ptr()], dims=(gate.numel(),), variant=variant)
    return out


def _unary(op: str, x: torch.Tensor, out: torch.Tensor | None, variant: int) -> torch.Tensor:
    _check(x, "x")
    out = torch.empty_like(x) if out is None else out
    _check(out, "out", x.dtype)
    if out.numel() != x.numel():
        raise ValueError(f"{op}: out has {out.numel()} elements, x has {x.numel()}")
    _run(op, x, [x.data_ptr(), out.data_ptr()], dims=(x.numel(),), variant=variant)
    return out


@_tensor_device
def relu(x: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``y = max(x, 0)``; values <= 0 map to +0 and NaN propagates (tasks/relu/reference.py, ``reference``)."""
    return _unary("relu", x, out, variant)


@_tensor_device
def sigmoid(x: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``y = 1 / (1 + exp(-x))`` (tasks/sigmoid/reference.py, ``reference``)."""
    return _unary("sigmoid", x, out, variant)


@_tensor_device
def sigmoid_shift(x: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``y = sigmoid(x) + 1`` (tasks/sigmoid_shift/reference.py, ``reference``)."""
    return _unary("sigmoid_shift", x, out, variant)


@_tensor_device
def lion(p: torch.Tensor, g: torch.Tensor, m: torch.Tensor, lr: float = 1e-3, wd: float = 0.1, beta1: float = 0.9,
         beta2: float = 0.99, p_out: torch.Tensor | None = None, m_out: torch.Tensor | None = None,
         variant: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """One Lion step (tasks/lion/reference.py, ``reference``; defaults from tasks/lion/opspec.json attrs):
    ``c = beta1*m + (1-beta1)*g``, ``p_out = p*(1 - lr*wd) - lr*sign(c)``, ``m_out = beta2*m + (1-beta2)*g``.
    Returns ``(p_out, m_out)``."""
    _check(p, "p")
    _check(g, "g", p.dtype)
    _check(m, "m", p.dtype)
    if g.numel() != p.numel() or m.numel() != p.numel():
        raise ValueError("p, g and m must have the same number of elements")
    p_out = torch.empty_like(p) if p_out is None else p_out
    m_out = torch.empty_like(p) if m_out is None else m_out
    _check(p_out, "p_out", p.dtype)
    _check(m_out, "m_out", p.dtype)
    _run("lion", p, [p.data_ptr(), g.data_ptr(), m.data_ptr(), p_out.data_ptr(), m_out.data_ptr()], dims=(p.numel(),),
         attrs=(float(lr), float(wd), float(beta1), float(beta2)), variant=variant)
    return p_out, m_out


@_tensor_device
def gemv(a: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``y[r] = sum_k A[r, k] * x[k]`` with A ``[M, K]`` row-major (tasks/gemv/reference.py, ``reference``)."""
    _check(a, "A")
    _check(x, "x", a.dtype)
    if a.dim() != 2 or x.numel() != a.shape[1]:
        raise ValueError(f"gemv needs A [M,K] and x [K], got {tuple(a.shape)} and {tuple(x.shape)}")
    m, k = a.shape
    out = torch.empty((m,), dtype=a.dtype, device=a.device) if out is None else out
    _check(out, "out", a.dtype)
    _run("gemv", a, [a.data_ptr(), x.data_ptr(), out.data_ptr()], dims=(m, k), variant=variant)
    return out


@_tensor_device
def softmax(x: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """Row softmax over the last axis (tasks/softmax/reference.py:104-106)."""
    _check(x, "x")
    n = x.shape[-1]
    m = x.numel() // max(n, 1)
    out = torch.empty_like(x) if out is None else out
    _check(out, "out", x.dtype)
    _run("softmax", x, [x.data_ptr(), out.data_ptr()], dims=(m, n), variant=variant)
    return out


@_tensor_device
def reduction_sum(x: torch.Tensor, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """Row sum over the last axis (tasks/reduction_sum/reference.py:104-106)."""
    _check(x, "x")
    n = x.shape[-1]
    m = x.numel() // max(n, 1)
    out = torch.empty(x.shape[:-1], dtype=x.dtype, device=x.device) if out is None else out
    _check(out, "out", x.dtype)
    _run("reduction_sum", x, [x.data_ptr(), out.data_ptr()], dims=(m, n), variant=variant)
    return out


@_tensor_device
def rope(x: torch.Tensor, base: float = 10000.0, out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """Rotate-half RoPE over ``[B, H, S, D]`` (tasks/rope/reference.py:105-115)."""
    _check(x, "x")
    if x.dim() != 4:
        raise ValueError("rope expects x [B, H, S, D]")
    b, h, s, d = x.shape
    out = torch.empty_like(x) if out is None else out
    _check(out, "out", x.dtype)
    _run("rope", x, [x.data_ptr(), out.data_ptr()], dims=(b, h, s, d), attrs=(base,), variant=variant)
    return out


@_tensor_device
def bitdelta_gemm(x: torch.Tensor, bits: torch.Tensor, scale: float = 0.02, out: torch.Tensor | None = None,
                  variant: int = 0) -> torch.Tensor:
    """``y = scale * x @ W`` with W ``[K, N]`` of +-1 from ``bits [K/32, N]`` (int32/uint32 words;
    bit j of ``bits[kb, n]`` is ``W[kb*32 + j, n]``, set = +1) — tasks/bitdelta_gemm/reference.py:99-130."""
    _check(x, "x")
    _check(bits, "bits")
    if bits.element_size() != 4:
        raise TypeError("bits must hold 32-bit words")
    m, k = x.shape
    kb, n = bits.shape
    if kb * 32 != k:
        raise ValueError(f"bits has {kb} word rows, expected K/32 = {k // 32}")
    out = torch.empty((m, n), dtype=x.dtype, device=x.device) if out is None else out
    _check(out, "out", x.dtype)
    _run("bitdelta_gemm", x, [x.data_ptr(), bits.data_ptr(), out.data_ptr()], dims=(m, n, k), attrs=(scale,), variant=variant)
    return out


@_tensor_device
def bitdelta_gemm_base(x: torch.Tensor, w_base: torch.Tensor, s_words: torch.Tensor, alpha: torch.Tensor,
                       out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``y = x @ (W_base + diag(alpha) S)^T`` with S in {-1,+1} packed along K as ``s_words [N, K/32]``."""
    _check(x, "x")
    _check(w_base, "w_base", x.dtype)
    _check(s_words, "s_words")
    _check(alpha, "alpha", x.dtype)
    m, k = x.shape
    n = w_base.shape[0]
    if w_base.shape[1] != k or s_words.shape != (n, k // 32) or alpha.numel() != n:
        raise ValueError("bitdelta_gemm_base: inconsistent shapes")
    out = torch.empty((m, n), dtype=x.dtype, device=x.device) if out is None else out
    _check(out, "out", x.dtype)
    _run("bitdelta_gemm_base", x, [x.data_ptr(), w_base.data_ptr(), s_words.data_ptr(), alpha.data_ptr(), out.data_ptr()],
         dims=(m, n, k), variant=variant)
    return out


@_tensor_device
def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, causal: bool = False,
                    out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """``softmax(q k^T * scale [+ causal mask]) v`` over ``[B, H, S, D]``
    (tasks/flash_attention/reference.py:113-119; the causal mask keeps key j <= query i)."""
    _check(q, "q")
    _check(k, "k", q.dtype)
    _check(v, "v", q.dtype)
    if q.dim() != 4 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError("flash_attention expects q, k, v of the same shape [B, H, S, D]")
    b, h, s, d = q.shape
    out = torch.empty_like(q) if out is None else out
    _check(out, "out", q.dtype)
    _run("flash_attention", q, [q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()], dims=(b, h, s, d), attrs=(scale,),
         variant=variant, flags=1 if causal else 0)
    return out


@_tensor_device
def varlen_kda(q, k, v, g, beta, a_log, dt_bias, initial_state, cu_seqlens, scale, lower_bound: float = -5.0,
               output: torch.Tensor | None = None, final_state: torch.Tensor | None = None, variant: int = 0,
               workspace: torch.Tensor | None = None):
    """Packed-varlen KDA forward (tasks/varlen_kda/reference.py:323-374).  ``scale`` is the
    task's one-element fp32 tensor; returns ``(output [T,H,D], final_state [N,H,D,D])``.
    ``variant``: 0 = the two-pass kernels over ``workspace`` (uint8, at least
    ``varlen_kda_workspace_bytes``; allocated here when not given) where they apply (D = 128),
    else the 16-token chunked kernel (D = 128), else the recurrent one; 4 = two-pass only;
    1 = 16-token chunked only; 2 = recurrent only."""
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        _check(t, name, q.dtype)
    for name, t in (("A_log", a_log), ("dt_bias", dt_bias), ("initial_state", initial_state), ("scale", scale)):
        _check(t, name, torch.float32)
    _check(cu_seqlens, "cu_seqlens", torch.int32)
    t_, h, d = q.shape
    n = cu_seqlens.numel() - 1
    output = torch.empty_like(v) if output is None else output
    final_state = torch.empty((n, h, d, d), dtype=torch.float32, device=q.device) if final_state is None else final_state
    need = varlen_kda_workspace_bytes(t_, n, h, d) if variant in (0, 4) and n > 0 else 0
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else 0
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    ptrs = [x.data_ptr() for x in (q, k, v, g, beta, a_log, dt_bias, initial_state, cu_seqlens, scale, output, final_state)]
    _run("varlen_kda", q, ptrs + [ws_ptr], dims=(n, h, d, t_, ws_bytes), attrs=(lower_bound,), variant=variant)
    return output, final_state


def varlen_kda_workspace_bytes(total_tokens: int, num_seqs: int, heads: int, dim: int) -> int:
    """Workspace bytes of the two-pass varlen KDA kernels (0 when they do not apply)."""
    return int(_native.load().sf_varlen_kda_workspace_bytes(total_tokens, num_seqs, heads, dim))


@_tensor_device
def kda(q, k, v, g, beta, a_log, dt_bias, initial_state, scale, lower_bound: float = -5.0,
        output: torch.Tensor | None = None, final_state: torch.Tensor | None = None,
        work_items: torch.Tensor | None = None, item_counts: torch.Tensor | None = None,
        handoff_states: torch.Tensor | None = None, variant: int = 0):
    """Fixed-length KDA forward (tasks/kda/reference.py ``reference``): the varlen recurrence over
    one sequence of N tokens.  q, k, v, g ``[N, H, D]``, beta ``[N, H]``; A_log ``[H]``, dt_bias
    ``[H*D]``, initial_state ``[H, D, D]`` and the one-element ``scale`` in fp32.  The task's
    candidate-owned outputs (``work_items`` u32 ``[3, 2]`` as int32, ``item_counts`` ``[1]``,
    ``handoff_states`` ``[2, H, D, D]``) are allocated when not given; the work list is written,
    the hand-off states are not (one piece).  ``variant`` 0/2 run the recurrent fp32 kernel (the
    default at every D), 1 forces the chunked tensor-core kernel (D = 128).  Returns
    ``(output [N,H,D], final_state [H,D,D])``."""
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        _check(t, name, q.dtype)
    for name, t in (("A_log", a_log), ("dt_bias", dt_bias), ("initial_state", initial_state), ("scale", scale)):
        _check(t, name, torch.float32)
    n, h, d = q.shape
    dev = q.device
    output = torch.empty_like(v) if output is None else output
    final_state = torch.empty((h, d, d), dtype=torch.float32, device=dev) if final_state is None else final_state
    work_items = torch.empty((3, 2), dtype=torch.int32, device=dev) if work_items is None else work_items
    item_counts = torch.empty((1,), dtype=torch.int32, device=dev) if item_counts is None else item_counts
    handoff_states = torch.empty((2, h, d, d), dtype=torch.float32, device=dev) if handoff_states is None else handoff_states
    ptrs = [x.data_ptr() for x in (q, k, v, g, beta, a_log, dt_bias, initial_state, scale, output, final_state, work_items,
                                   item_counts, handoff_states)]
    _run("kda", q, ptrs, dims=(n, h, d), attrs=(lower_bound,), variant=variant)
    return output, final_state


@_tensor_device
def varlen_kda_gated(q, k, v, g, beta, cu_seqlens, scale: float, initial_state: torch.Tensor | None = None,
                     output: torch.Tensor | None = None, final_state: torch.Tensor | None = None, variant: int = 0,
                     workspace: torch.Tensor | None = None):
    """Gated KDA workload: q, k pre-normalised, ``g`` fp32 log-decay used directly, ``beta`` fp32
    gate used directly, state from zero (or ``initial_state``).

    At D = 128 the default (and ``variant=4``) runs the two-pass kernels over ``workspace`` (uint8,
    at least ``varlen_kda_gated_workspace_bytes``; allocated here when not given); ``variant=1``
    forces the single-pass 32-token kernel, 2 the recurrent kernel, 3 the 16-token kernel."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(t, name, q.dtype)
    _check(g, "g", torch.float32)
    _check(beta, "beta", torch.float32)
    _check(cu_seqlens, "cu_seqlens", torch.int32)
    t_, h, d = q.shape
    n = cu_seqlens.numel() - 1
    output = torch.empty_like(v) if output is None else output
    final_state = torch.empty((n, h, d, d), dtype=torch.float32, device=q.device) if final_state is None else final_state
    s0 = 0
    if initial_state is not None:
        _check(initial_state, "initial_state", torch.float32)
        s0 = initial_state.data_ptr()
    need = varlen_kda_gated_workspace_bytes(t_, n, h, d) if variant in (0, 4) else 0
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else 0
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    ptrs = [q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), cu_seqlens.data_ptr(), s0,
            output.data_ptr(), final_state.data_ptr(), ws_ptr]
    _run("varlen_kda_gated", q, ptrs, dims=(n, h, d, t_, ws_bytes), attrs=(scale,), variant=variant)
    return output, final_state


def varlen_kda_gated_workspace_bytes(total_tokens: int, num_seqs: int, heads: int, dim: int) -> int:
    """Workspace bytes of the two-pass gated KDA kernels (0 when they do not apply)."""
    return int(_native.load().sf_varlen_kda_gated_workspace_bytes(total_tokens, num_seqs, heads, dim))


@_tensor_device
def mamba2_chunk_scan(x, dt, dA_cumsum, b_mat, c_mat, d_skip, states, out: torch.Tensor | None = None,
                      variant: int = 0) -> torch.Tensor:
    """Mamba-2 SSD chunk scan of one B/C group (tasks/mamba2_chunk_scan/reference.py:106-127).

    x [B,L,H,P], dt [B,L,H], dA_cumsum [B,H,NC,CHUNK], b_mat/c_mat [B,L,N], d_skip [H],
    states [B,NC,H,P,N], all of one 16-bit dtype; returns y [B,L,H,P]."""
    tensors = (("x", x), ("dt", dt), ("dA_cumsum", dA_cumsum), ("Bmat", b_mat), ("Cmat", c_mat), ("Dskip", d_skip),
               ("states", states))
    for name, t in tensors:
        _check(t, name, x.dtype)
    if x.dim() != 4 or dA_cumsum.dim() != 4 or states.dim() != 5:
        raise ValueError("mamba2_chunk_scan expects x [B,L,H,P], dA_cumsum [B,H,NC,CHUNK], states [B,NC,H,P,N]")
    bsz, seq, heads, hd = x.shape
    nc, chunk = dA_cumsum.shape[2], dA_cumsum.shape[3]
    n = b_mat.shape[-1]
    want = {"dt": (bsz, seq, heads), "dA_cumsum": (bsz, heads, nc, chunk), "Bmat": (bsz, seq, n), "Cmat": (bsz, seq, n),
            "Dskip": (heads,), "states": (bsz, nc, heads, hd, n)}
    for name, t in tensors[1:]:
        if tuple(t.shape) != want[name]:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {want[name]}")
    if nc * chunk != seq:
        raise ValueError(f"SEQLEN {seq} != NCHUNKS {nc} * CHUNK {chunk}")
    out = torch.empty_like(x) if out is None else out
    _check(out, "out", x.dtype)
    ptrs = [t.data_ptr() for _, t in tensors] + [out.data_ptr()]
    _run("mamba2_chunk_scan", x, ptrs, dims=(bsz, seq, heads, hd, n, chunk), variant=variant)
    return out


# ---- serving operators: [tokens, heads, D] tensors with any token and head strides -----------------
#
# A decoding step makes these calls once a layer on a few tokens, so their host time counts: each tensor
# is looked at once, and the arguments go down in one packed struct.


def _gpu(t: torch.Tensor, name: str, dev: int | None = None) -> int:
    """The index of the GPU ``t`` is on; refused on the CPU or when it is not GPU ``dev``."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if dev is not None and index != dev:
        raise ValueError(f"tensors on more than one device (cuda:{dev}, {name} on cuda:{index})")
    return index


def _check_rows(t: torch.Tensor, name: str, dev: int | None = None, dtype: torch.dtype | None = None, shape=None,
                written: bool = False) -> tuple[int, int]:
    """Check a [tokens, heads, D] CUDA tensor with unit stride along D; return its token and head
    strides in elements (0 along an axis of one entry, whose stride says nothing)."""
    _gpu(t, name, dev)
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    size = t.shape
    if len(size) != 3:
        raise ValueError(f"{name} must have three axes (tokens, heads, D), got shape {tuple(size)}")
    if shape is not None and size != shape:
        raise ValueError(f"{name} has shape {tuple(size)}, expected {tuple(shape)}")
    n, h, d = size
    a, b, c = t.stride()
    if d > 1 and c != 1:
        raise ValueError(f"{name} must have unit stride along its last axis")
    if n <= 1:
        a = 0
    if h <= 1:
        b = 0
    if written and n * h:
        # Rows that share memory would be written by two threads: the axis with the larger stride has
        # to step over all that the other spans.
        near, far = ((a, n), (b, h)) if (a <= b and n > 1) or h <= 1 else ((b, h), (a, n))
        span = near[0] * (near[1] - 1) + d
        if (near[1] > 1 and near[0] < d) or (far[1] > 1 and far[0] < span):
            raise ValueError(f"{name} has rows that overlap (strides {t.stride()})")
    return a, b


def _check_vector(t: torch.Tensor, name: str, dev: int, dtype: torch.dtype, length: int | None = None) -> None:
    """Check a contiguous one-axis tensor of ``length`` entries."""
    _gpu(t, name, dev)
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.dim() != 1 or (length is not None and t.shape[0] != length) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with one axis{'' if length is None else f' of {length}'}, got shape {tuple(t.shape)}")


def _count(x: int, name: str) -> int:
    x = operator.index(x)
    if not 0 <= x < 1 << 63:
        raise ValueError(f"{name} must be >= 0 and below 2^63, got {x}")
    return x


def _workspace_bytes(t: torch.Tensor, dev: int) -> int:
    _gpu(t, "workspace", dev)
    if not t.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return t.numel() * t.element_size()


def _launch(name: str, dev: int, *fields) -> None:
    """Call a serving entry point on GPU ``dev``'s current stream, with that GPU current (the C ABI
    launches on the thread's current device); entering it costs more than the launch, so only if need be.
    The stream comes as the raw handle: a ``torch.cuda.Stream`` object would cost 3 us of a 12 us call."""
    if torch.cuda.current_device() == dev:
        _native.call_args(name, torch._C._cuda_getCurrentRawStream(dev), *fields)
    else:
        with torch.cuda.device(dev):
            _native.call_args(name, torch._C._cuda_getCurrentRawStream(dev), *fields)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                 base: float = 10000.0, eps: float = 1e-6, rotary_dim: int | None = None, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None, variant: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-head RMS norm of queries ``q [T, Hq, D]`` and keys ``k [T, Hk, D]`` (weights ``[D]``) and the
    rotate-half rotary embedding of their first ``rotary_dim`` (default D) elements at ``positions [T]``
    (int32), in one pass; :func:`rmsnorm` then :func:`rope`, at any positions.  ``q`` and ``k`` may be
    views of a packed projection (unit stride along D); ``q_out`` / ``k_out`` may be ``q`` / ``k``
    themselves (in place), otherwise they must not overlap the inputs.  ``variant``: 0 = by shape, 1 =
    vectorised (refused where it does not apply), 2 = general.  Returns ``(q_out, k_out)``."""
    dev = _gpu(q, "q")
    dtype = q.dtype
    qs, ks = _check_rows(q, "q", dev), _check_rows(k, "k", dev, dtype)
    t, hq, d = q.shape
    hk = k.shape[1]
    if k.shape[0] != t or k.shape[2] != d:
        raise ValueError(f"k has shape {tuple(k.shape)}, expected [{t}, heads, {d}]")
    _check_vector(q_weight, "q_weight", dev, dtype, d)
    _check_vector(k_weight, "k_weight", dev, dtype, d)
    _check_vector(positions, "positions", dev, torch.int32, t)
    if q_out is None:
        q_out, qos = q.new_empty(t, hq, d), (hq * d, d)
    else:
        qos = _check_rows(q_out, "q_out", dev, dtype, q.shape, written=True)
    if k_out is None:
        k_out, kos = k.new_empty(t, hk, d), (hk * d, d)
    else:
        kos = _check_rows(k_out, "k_out", dev, dtype, k.shape, written=True)
    _launch("sf_qk_norm_rope", dev, q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(),
            q_out.data_ptr(), k_out.data_ptr(), t, hq, hk, d, d if rotary_dim is None else rotary_dim, *qs, *ks, *qos, *kos, base, eps,
            _native.DTYPE_CODES[dtype_name(q)], variant)
    return q_out, k_out


def kv4_cache(num_pages: int, page_size: int, heads: int, dim: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """A zeroed 4-bit paged key/value cache for :func:`kv4_store`, :func:`kv4_load` and
    :func:`kv4_attention`: uint8 ``[num_pages, heads, page_size / 16, 18 * dim]``, 4.5 bits a value
    (``dim`` 64 or 128, ``page_size`` a multiple of 16).  Slot ``s`` is row ``s % page_size`` of page
    ``s // page_size``."""
    if page_size < 16 or page_size % 16 or dim not in (64, 128) or num_pages < 0 or heads < 1:
        raise ValueError("kv4_cache needs a page size that is a multiple of 16, dim 64 or 128 and at least one head")
    return torch.zeros((num_pages, heads, page_size // 16, 18 * dim), dtype=torch.uint8, device=device)


def _check_cache(cache: torch.Tensor, dev: int | None = None) -> tuple[int, int, int, int]:
    """(pages, heads, page size, D) of a 4-bit cache."""
    _gpu(cache, "cache", dev)
    if cache.dtype != torch.uint8:
        raise TypeError(f"cache has dtype {cache.dtype}, expected torch.uint8")
    if cache.dim() != 4 or cache.shape[3] not in (18 * 64, 18 * 128) or cache.shape[2] < 1 or not cache.is_contiguous():
        raise ValueError(f"cache must be a contiguous [pages, heads, page_size / 16, 18 * D], D 64 or 128, got {tuple(cache.shape)}")
    pages, heads, tiles, record = cache.shape
    return pages, heads, 16 * tiles, record // 18


def kv4_store(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: torch.Tensor) -> torch.Tensor:
    """Quantise the tokens ``k, v [T, H, D]`` (unit stride along D) to 4 bits and write them at ``slots
    [T]`` (int32) of ``cache`` (:func:`kv4_cache`); returns ``cache``.  Every 64 elements of a token's
    head get a bf16 minimum and scale = (max - min) / 15 and codes rint((x - minimum) / scale) in 0..15, in
    fp32 operations; a group that is not finite reads back as NaN.  A negative slot is padding and skipped, one past the
    cache is skipped and reported by :func:`kernel_status` (code 3).  The slots must differ."""
    dev = _gpu(k, "k")
    pages, heads, page, d = _check_cache(cache, dev)
    t = k.shape[0] if k.dim() else 0
    ks, vs = _check_rows(k, "k", dev, None, (t, heads, d)), _check_rows(v, "v", dev, k.dtype, (t, heads, d))
    _check_vector(slots, "slots", dev, torch.int32, t)
    _launch("sf_kv4_store", dev, k.data_ptr(), v.data_ptr(), slots.data_ptr(), cache.data_ptr(), t, heads, d, pages, page, *ks, *vs,
            _native.DTYPE_CODES[dtype_name(k)], 0)
    return cache


def kv4_load(cache: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16, k_out: torch.Tensor | None = None,
             v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Read the tokens at ``slots [T]`` (int32, in any order, repeated or not) of a 4-bit cache back as
    ``(k, v)``, each ``[T, H, D]`` in ``dtype`` (minimum + scale * code, rounded once; the minimum is a bf16, so fp16
    values within 2^8 of the type's largest may come back infinite), e.g. as the
    context of a prompt's next chunk for :func:`window_attention`.  Negative slots (and, reported by
    :func:`kernel_status`, slots past the cache) read as zeros.  ``k_out`` / ``v_out`` set the type when
    given."""
    dev = _gpu(cache, "cache")
    pages, heads, page, d = _check_cache(cache)
    _check_vector(slots, "slots", dev, torch.int32)
    shape = (slots.shape[0], heads, d)
    given = k_out if k_out is not None else v_out
    dtype = dtype if given is None else given.dtype
    if k_out is None:
        k_out, ks = cache.new_empty(*shape, dtype=dtype), (heads * d, d)
    else:
        ks = _check_rows(k_out, "k_out", dev, dtype, shape, written=True)
    if v_out is None:
        v_out, vs = cache.new_empty(*shape, dtype=dtype), (heads * d, d)
    else:
        vs = _check_rows(v_out, "v_out", dev, dtype, shape, written=True)
    _launch("sf_kv4_load", dev, k_out.data_ptr(), v_out.data_ptr(), slots.data_ptr(), cache.data_ptr(), *shape, pages, page, *ks, *vs,
            _native.DTYPE_CODES[dtype_name(k_out)], 0)
    return k_out, v_out


def kv4_attention_workspace_bytes(batch: int, q_heads: int, kv_heads: int, dim: int, page_size: int, table_width: int, window: int = 0,
                                  sinks: int = 0, variant: int = 0) -> int:
    """Workspace bytes of :func:`kv4_attention` (0 when a request's keys stay with one CTA)."""
    return int(_native.load().sf_kv4_attention_workspace_bytes(batch, q_heads, kv_heads, dim, page_size, table_width, window, sinks, variant))


@functools.lru_cache(maxsize=512)
def _kv4_attention_need(dev: int, *sizes: int) -> int:
    """The sizes' workspace bytes on GPU ``dev`` (the plan goes by its SMs, so it is asked for with that GPU current):
    a decode loop asks for the same ones again and again."""
    with torch.cuda.device(dev):
        return kv4_attention_workspace_bytes(*sizes)


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, scale: float, window: int = 0,
                  sinks: int = 0, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """Attention of one query token a request over the 4-bit paged cache: ``softmax(q K^T * scale) V``.

    ``q [B, Hq, D]`` (unit stride along D), Hq a multiple of the cache's heads; ``block_table [B, width]``
    (int32, rows may be strided) holds each request's pages in order, ``seq_lens [B]`` (int32) its tokens
    in the cache, the query's own last.  Token ``j`` is seen when ``j >= seq_len - window`` or ``j <
    sinks`` (``window`` 0: all).  A length of 0 gives zeros; a length past the table is cut to it and a
    page id outside the cache hides its tokens, both reported by :func:`kernel_status` (code 3); a request
    with every token hidden gives zeros.  Softmax in fp32, its weights to 11 (bf16) or 22 (fp16) bits in their
    product.  q and ``out`` need 16-byte aligned rows and must not overlap.
    ``workspace`` (uint8, :func:`kv4_attention_workspace_bytes`) is allocated here when not given;
    calls that overlap on the GPU need one each.  ``variant``: 0 = by size, 1 = all requests' keys
    dealt evenly to all CTAs, 3 = a CTA a (request, head)."""
    dev = _gpu(q, "q")
    window, sinks = _count(window, "window"), _count(sinks, "sinks")
    dtype = q.dtype
    pages, heads, page, d = _check_cache(cache, dev)
    qs = _check_rows(q, "q", dev)
    b, hq, qd = q.shape
    if qd != d or heads == 0 or hq % heads:
        raise ValueError(f"q must be [B, a multiple of {heads}, {d}] for this cache, got {tuple(q.shape)}")
    _gpu(block_table, "block_table", dev)
    if block_table.dtype != torch.int32:
        raise TypeError(f"block_table has dtype {block_table.dtype}, expected torch.int32")
    if block_table.dim() != 2 or block_table.shape[0] != b or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be [{b}, width] with unit stride along a row")
    width = block_table.shape[1]
    _check_vector(seq_lens, "seq_lens", dev, torch.int32, b)
    if out is None:
        out, os_ = q.new_empty(b, hq, d), (hq * d, d)
    else:
        os_ = _check_rows(out, "out", dev, dtype, q.shape, written=True)
    if workspace is None:
        need = _kv4_attention_need(dev, b, hq, heads, d, page, width, window, sinks, variant)
        if need:
            workspace = cache.new_empty(need)
    else:
        need = _workspace_bytes(workspace, dev)
    _launch("sf_kv4_attention", dev, q.data_ptr(), cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
            0 if workspace is None else workspace.data_ptr(), need, b, hq, heads, d, pages, page, width,
            block_table.stride(0) if b > 1 else 0, *qs, *os_, window, sinks, scale, _native.DTYPE_CODES[dtype_name(q)], variant)
    return out


def window_attention_workspace_bytes(q_tokens: int, k_tokens: int, sequences: int, q_heads: int, kv_heads: int, dim: int, window: int = 0,
                                     sinks: int = 0) -> int:
    """Workspace bytes of :func:`window_attention` (0 when the keys of a row tile stay with one CTA)."""
    return int(_native.load().sf_window_attention_workspace_bytes(q_tokens, k_tokens, sequences, q_heads, kv_heads, dim, window, sinks))


@functools.lru_cache(maxsize=512)
def _window_attention_need(dev: int, *sizes: int) -> int:
    with torch.cuda.device(dev):  # as above
        return window_attention_workspace_bytes(*sizes)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, scale: float, window: int = 0, sinks: int = 0,
                     cu_seqlens_k: torch.Tensor | None = None, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                     variant: int = 0) -> torch.Tensor:
    """Causal attention of packed prompts with grouped heads, a sliding window and sinks.

    ``q [Tq, Hq, D]``, ``k, v [Tk, Hk, D]`` (unit stride along D, Hq a multiple of Hk); sequence ``s`` has
    the queries ``cu_seqlens[s] : cu_seqlens[s + 1]`` and the keys of ``cu_seqlens_k`` (default: the same
    rows).  Query ``i`` of a sequence with nq queries and nk keys sits at ``p = i + nk - nq`` and sees the
    keys ``j <= p`` with ``j > p - window`` or ``j < sinks`` (``window`` 0: all ``j <= p``), so a prompt's next
    chunk comes with its whole context as keys.  A query that sees nothing gives zeros; rows of ``out``
    that belong to no sequence are left as they were (with no ``out`` given: not initialised).  ``out`` must not
    overlap the inputs.  Softmax in fp32, its
    weights to some 16 (bf16) or 22 (fp16) bits in their product.  D up to 256; D 64 and 128 with 16-byte aligned rows and at most 128 query heads a key head run on the tensor cores, where few queries with many keys
    are split over the keys by way of ``workspace`` (uint8, :func:`window_attention_workspace_bytes`,
    allocated here when not given; calls that overlap on the GPU need one each).  ``variant``: 0 = by
    shape, 1 = tensor cores (refused where they do not apply), 2 = general kernel, 4 = unsplit."""
    dev = _gpu(q, "q")
    window, sinks = _count(window, "window"), _count(sinks, "sinks")
    dtype = q.dtype
    qs, ks = _check_rows(q, "q", dev), _check_rows(k, "k", dev, dtype)
    vs = _check_rows(v, "v", dev, dtype, k.shape)
    tq, hq, d = q.shape
    tk, hk, kd = k.shape
    if kd != d or hk == 0 or hq % hk:
        raise ValueError(f"window_attention expects k and v [Tk, Hk, {d}] with Hk dividing {hq}, got {tuple(k.shape)}")
    _check_vector(cu_seqlens, "cu_seqlens", dev, torch.int32)
    seqs = cu_seqlens.shape[0] - 1
    if seqs < 0:
        raise ValueError("cu_seqlens must have at least one entry")
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens
        if tk != tq:
            raise ValueError(f"k has {tk} rows and q {tq}: cu_seqlens_k is needed")
    else:
        _check_vector(cu_seqlens_k, "cu_seqlens_k", dev, torch.int32, seqs + 1)
    if out is None:
        out, os_ = q.new_empty(tq, hq, d), (hq * d, d)
    else:
        os_ = _check_rows(out, "out", dev, dtype, q.shape, written=True)
    if workspace is None:
        need = 0 if variant in (2, 4) else _window_attention_need(dev, tq, tk, seqs, hq, hk, d, window, sinks)
        if need:
            workspace = q.new_empty(need, dtype=torch.uint8)
    else:
        need = _workspace_bytes(workspace, dev)
    _launch("sf_window_attention", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens.data_ptr(), cu_seqlens_k.data_ptr(),
            out.data_ptr(), 0 if workspace is None else workspace.data_ptr(), need, tq, tk, seqs, hq, hk, d, *qs, *ks, *vs, *os_, window, sinks, scale, _native.DTYPE_CODES[dtype_name(q)], variant)
    return out
