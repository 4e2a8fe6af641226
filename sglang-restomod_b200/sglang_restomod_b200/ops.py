"""Torch-facing wrappers of the libb200moe C ABI.

Every function here takes CUDA tensors, validates what the C ABI cannot see
(dtype, device, contiguity), and calls the library on the current CUDA stream.
Outputs are allocated here unless the caller passes them (the reference's
``Tensor(a!) out`` convention, ``quant/sm70_fp8_moe/shim.cpp:50-56``).

Workspaces are cached per device, sized once and zero-filled; a call that
needs a larger one grows it, except during CUDA-graph capture, where growing
would be an allocation inside the capture and raises instead (size them up
front with :func:`reserve_workspace`, as the reference sizes its decode
workspace for the largest capture batch, ``decode_gemv.py:170-180``).
"""

from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib

_DTYPE_CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_WS_LOCK = threading.Lock()
_WORKSPACES: dict[int, torch.Tensor] = {}


def _vp(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _code(t: torch.Tensor, what: str) -> int:
    try:
        return _DTYPE_CODE[t.dtype]
    except KeyError:
        raise TypeError(f"{what} must be bf16 or f16, got {t.dtype}") from None


def _cuda(t: torch.Tensor, what: str) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{what} must be a CUDA tensor")


def _contig(t: torch.Tensor, what: str) -> None:
    _cuda(t, what)
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def lib():
    return _lib._LIB or _lib.load()


def num_sms() -> int:
    return int(lib().b200_num_sms())


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Per-device zero-filled workspace of at least ``nbytes`` bytes."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    with _WS_LOCK:
        ws = _WORKSPACES.get(index)
        if ws is not None and ws.numel() >= nbytes:
            return ws
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(
                f"b200 workspace needs {nbytes} bytes during CUDA-graph capture; "
                "call reserve_workspace() before capturing"
            )
        size = max(nbytes, 0 if ws is None else ws.numel())
        ws = torch.zeros(size + 256, dtype=torch.uint8, device=torch.device("cuda", index))
        # The library wants a 256-byte aligned base.
        offset = (-ws.data_ptr()) % 256
        ws = ws[offset : offset + size]
        _WORKSPACES[index] = ws
        return ws


def reserve_workspace(nbytes: int, device: torch.device | None = None) -> torch.Tensor:
    return workspace(nbytes, device or torch.device("cuda", torch.cuda.current_device()))


def workspace_status(device: torch.device | None = None, reset: bool = True) -> int:
    """Device error bits recorded by the kernels (0 = none). Synchronizes."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    ws = _WORKSPACES.get(device.index if device.index is not None else torch.cuda.current_device())
    if ws is None:
        return 0
    bits = ctypes.c_int32(0)
    _lib.check(lib().b200_workspace_status(_vp(ws), ctypes.byref(bits), int(reset), _stream(ws.device)))
    return int(bits.value)


# ----------------------------------------------------------------- routing
def align_capacity(numel: int, num_experts: int, block_size: int) -> tuple[int, int]:
    cap = numel + min(numel, num_experts) * (block_size - 1)
    return cap, (cap + block_size - 1) // block_size


def moe_align_block_size(topk_ids: torch.Tensor, block_size: int, num_experts: int, out=None):
    """(sorted_token_ids, expert_ids, num_tokens_post_pad) for ``topk_ids``."""
    _contig(topk_ids, "topk_ids")
    if topk_ids.dtype != torch.int32:
        raise TypeError(f"topk_ids must be int32, got {topk_ids.dtype}")
    numel = topk_ids.numel()
    cap, blocks = align_capacity(numel, num_experts, block_size)
    if out is None:
        dev = topk_ids.device
        sorted_ids = torch.empty(cap, dtype=torch.int32, device=dev)
        expert_ids = torch.empty(blocks, dtype=torch.int32, device=dev)
        ntpp = torch.empty(1, dtype=torch.int32, device=dev)
    else:
        sorted_ids, expert_ids, ntpp = out
    _lib.check(
        lib().b200_moe_align_block_size(
            _vp(topk_ids), numel, num_experts, block_size, _vp(sorted_ids), sorted_ids.numel(),
            _vp(expert_ids), expert_ids.numel(), _vp(ntpp), _stream(topk_ids.device),
        )
    )
    return sorted_ids, expert_ids, ntpp


# ----------------------------------------------------------------- combine
_LOGIT_CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16,
               torch.float32: _lib.DTYPE_F32}


def topk_route(router_logits: torch.Tensor, top_k: int, *, scoring: int = _lib.SCORING_SOFTMAX,
               renormalize: bool = True, correction_bias: torch.Tensor | None = None,
               out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """(topk_ids int32 [T, k], topk_weights fp32 [T, k]) from router logits [T, E]."""
    _contig(router_logits, "router_logits")
    try:
        code = _LOGIT_CODE[router_logits.dtype]
    except KeyError:
        raise TypeError(f"router_logits must be bf16, f16 or f32, got {router_logits.dtype}") from None
    tokens, experts = (int(d) for d in router_logits.shape)
    if correction_bias is not None:
        _contig(correction_bias, "correction_bias")
        if correction_bias.dtype != torch.float32 or correction_bias.numel() != experts:
            raise ValueError("correction_bias must be fp32 [num_experts]")
    if out is None:
        ids = torch.empty(tokens, top_k, dtype=torch.int32, device=router_logits.device)
        w = torch.empty(tokens, top_k, dtype=torch.float32, device=router_logits.device)
    else:
        ids, w = out
    _lib.check(
        lib().b200_topk_route(
            _vp(router_logits), code, tokens, experts, top_k, scoring, int(renormalize),
            _vp(correction_bias), _vp(ids), _vp(w), _stream(router_logits.device),
        )
    )
    return ids, w


def topk_route_grouped(router_logits: torch.Tensor, top_k: int, num_expert_group: int,
                       topk_group: int, *, scoring: int = _lib.SCORING_SOFTMAX,
                       renormalize: bool = True, correction_bias: torch.Tensor | None = None):
    """Grouped top-k (upstream grouped_topk / biased_grouped_topk): only the
    ``topk_group`` best of ``num_expert_group`` expert groups are selectable."""
    _contig(router_logits, "router_logits")
    try:
        code = _LOGIT_CODE[router_logits.dtype]
    except KeyError:
        raise TypeError(f"router_logits must be bf16, f16 or f32, got {router_logits.dtype}") from None
    tokens, experts = (int(d) for d in router_logits.shape)
    if correction_bias is not None:
        _contig(correction_bias, "correction_bias")
        if correction_bias.dtype != torch.float32 or correction_bias.numel() != experts:
            raise ValueError("correction_bias must be fp32 [num_experts]")
    ids = torch.empty(tokens, top_k, dtype=torch.int32, device=router_logits.device)
    w = torch.empty(tokens, top_k, dtype=torch.float32, device=router_logits.device)
    _lib.check(
        lib().b200_topk_route_grouped(
            _vp(router_logits), code, tokens, experts, top_k, scoring, int(renormalize),
            _vp(correction_bias), int(num_expert_group), int(topk_group), _vp(ids), _vp(w),
            _stream(router_logits.device),
        )
    )
    return ids, w


def append_shared_route(topk_ids: torch.Tensor, topk_weights: torch.Tensor, shared_id: int,
                        shared_weight: float = 1.0):
    """[T, k] routes -> [T, k + 1] with one route per token to ``shared_id``."""
    _contig(topk_ids, "topk_ids")
    _contig(topk_weights, "topk_weights")
    tokens, top_k = (int(d) for d in topk_ids.shape)
    ids = torch.empty(tokens, top_k + 1, dtype=torch.int32, device=topk_ids.device)
    w = torch.empty(tokens, top_k + 1, dtype=torch.float32, device=topk_ids.device)
    _lib.check(
        lib().b200_append_shared_route(_vp(topk_ids), _vp(topk_weights), tokens, top_k, shared_id,
                                       float(shared_weight), _vp(ids), _vp(w),
                                       _stream(topk_ids.device))
    )
    return ids, w


def moe_sum_reduce(input_tensor: torch.Tensor, output_tensor: torch.Tensor,
                   routed_scaling_factor: float = 1.0) -> torch.Tensor:
    """``out[t] = rsf * sum_k in[t, k]`` (``quant/sm70_fp4_moe/sum_reduce.py:84-123``)."""
    _contig(input_tensor, "input")
    _contig(output_tensor, "output")
    if input_tensor.dtype != output_tensor.dtype:
        raise ValueError(
            f"moe_sum_reduce dtype mismatch: input {input_tensor.dtype}, output {output_tensor.dtype}"
        )
    tokens, top_k, hidden = input_tensor.shape
    if tuple(output_tensor.shape) != (tokens, hidden):
        raise ValueError(f"output must be [{tokens}, {hidden}], got {tuple(output_tensor.shape)}")
    _lib.check(
        lib().b200_moe_sum_reduce(
            _vp(input_tensor), _vp(output_tensor), tokens, top_k, hidden,
            _code(input_tensor, "input"), float(routed_scaling_factor), _stream(input_tensor.device),
        )
    )
    return output_tensor


def moe_combine(routed: torch.Tensor, topk_ids: torch.Tensor | None, num_experts: int,
                routed_scaling_factor: float = 1.0, shared_out: torch.Tensor | None = None,
                out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16):
    """Sum weighted per-route rows ``routed [T*k, H]`` over valid slots."""
    _contig(routed, "routed")
    if topk_ids is None:
        raise ValueError("topk_ids is required to know top_k")
    _contig(topk_ids, "topk_ids")
    tokens, top_k = topk_ids.shape
    hidden = routed.shape[-1]
    if out is None:
        out = torch.empty(tokens, hidden, dtype=out_dtype, device=routed.device)
    if shared_out is not None:
        _contig(shared_out, "shared_out")
    _lib.check(
        lib().b200_moe_combine(
            _vp(routed), _code(routed, "routed"), _vp(topk_ids), num_experts, tokens, top_k, hidden,
            float(routed_scaling_factor), _vp(shared_out),
            _code(shared_out, "shared_out") if shared_out is not None else 0,
            _vp(out), _code(out, "out"), _stream(routed.device),
        )
    )
    return out


# ----------------------------------------------------------------- prepack
def fp8_prepack(w: torch.Tensor, gated: bool) -> torch.Tensor:
    """e4m3 ``[E, N, K]`` (or ``[N, K]``) -> streamed bank ``[E, N*K]`` uint8."""
    _contig(w, "weight")
    if w.dtype != torch.float8_e4m3fn:
        raise TypeError(f"weight must be float8_e4m3fn, got {w.dtype}")
    w3 = w.unsqueeze(0) if w.dim() == 2 else w
    e, n, k = (int(d) for d in w3.shape)
    nbytes = int(lib().b200_fp8_packed_bytes(e, n, k))
    out = torch.empty(e, nbytes // e, dtype=torch.uint8, device=w.device)
    _lib.check(lib().b200_fp8_prepack(_vp(w3), e, n, k, int(gated), _vp(out), _stream(w.device)))
    return out


def nvfp4_prepack(w: torch.Tensor, scales: torch.Tensor, gated: bool) -> torch.Tensor:
    """ModelOpt ``[E, N, K/2]`` uint8 + ``[E, N, K/16]`` e4m3 -> streamed bank."""
    _contig(w, "weight")
    _contig(scales, "scales")
    if w.dtype != torch.uint8:
        raise TypeError(f"packed NVFP4 weight must be uint8, got {w.dtype}")
    if scales.dtype != torch.float8_e4m3fn:
        raise TypeError(f"NVFP4 scales must be float8_e4m3fn, got {scales.dtype}")
    w3 = w.unsqueeze(0) if w.dim() == 2 else w
    s3 = scales.unsqueeze(0) if scales.dim() == 2 else scales
    e, n, half_k = (int(d) for d in w3.shape)
    k = 2 * half_k
    if tuple(s3.shape) != (e, n, k // 16):
        raise ValueError(f"scales must be [{e}, {n}, {k // 16}], got {tuple(s3.shape)}")
    nbytes = int(lib().b200_nvfp4_packed_bytes(e, n, k))
    if nbytes < 0:
        raise ValueError(f"NVFP4 bank needs N and K multiples of 128, got N={n} K={k}")
    out = torch.empty(e, nbytes // e, dtype=torch.uint8, device=w.device)
    _lib.check(
        lib().b200_nvfp4_prepack(_vp(w3), _vp(s3), e, n, k, int(gated), _vp(out), _stream(w.device))
    )
    return out


# ------------------------------------------------------------------- GEMMs
def gemm_workspace_bytes(convert_elems: int) -> int:
    return int(lib().b200_gemm_workspace_bytes(int(convert_elems)))


def linear(x: torch.Tensor, packed: torch.Tensor, n: int, *, quant: int,
           scales: torch.Tensor | None = None, global_scale: torch.Tensor | None = None,
           gated_mode: int = _lib.GATED_NONE, out: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None, loads_only: bool = False) -> torch.Tensor:
    """Dense ``y = x . dequant(W)^T`` on a prepacked bank (one expert).
    ``loads_only``: the call's data-movement floor (no math, ``out`` untouched)."""
    _contig(x, "x")
    x2 = x.reshape(-1, x.shape[-1])
    m, k = (int(d) for d in x2.shape)
    cols = n // 2 if gated_mode == _lib.GATED_FUSED else n
    if out is None:
        out = torch.empty(m, cols, dtype=out_dtype or x.dtype, device=x.device)
    ws = workspace(gemm_workspace_bytes(m * k if x.dtype == torch.bfloat16 else 0), x.device)
    fn = lib().b200_linear_loads_only if loads_only else lib().b200_linear
    _lib.check(
        fn(
            quant, _vp(x2), _code(x2, "x"), m, k, _vp(packed), _vp(scales), _vp(global_scale), n,
            gated_mode, _vp(out), _code(out, "out"), _vp(ws), ws.numel(), _stream(x.device),
        )
    )
    return out.reshape(*x.shape[:-1], cols)


def moe_gemm(a: torch.Tensor, packed: torch.Tensor, n: int, *, quant: int, num_experts: int,
             sorted_token_ids: torch.Tensor, expert_ids: torch.Tensor,
             num_tokens_post_pad: torch.Tensor, block_size: int, top_k: int, num_routes: int,
             c: torch.Tensor, scales: torch.Tensor | None = None,
             global_scale: torch.Tensor | None = None, topk_weights: torch.Tensor | None = None,
             mul_topk_weights: bool = False, gated_mode: int = _lib.GATED_NONE,
             loads_only: bool = False) -> torch.Tensor:
    """Grouped expert GEMM with ``moe_wna16_marlin_gemm`` routing semantics.
    ``loads_only``: the call's data-movement floor (no math, ``c`` untouched)."""
    _contig(a, "a")
    _contig(c, "c")
    a_rows, k = (int(d) for d in a.reshape(-1, a.shape[-1]).shape)
    if topk_weights is not None:
        _contig(topk_weights, "topk_weights")
        if topk_weights.dtype != torch.float32:
            topk_weights = topk_weights.float().contiguous()
    if c.shape[0] < num_routes:
        raise ValueError(f"c has {c.shape[0]} rows, the routes need {num_routes}")
    if mul_topk_weights and (topk_weights is None or topk_weights.numel() < num_routes):
        raise ValueError("mul_topk_weights needs one topk weight per route")
    groups = min(expert_ids.numel(), sorted_token_ids.numel() // block_size)
    ws = workspace(gemm_workspace_bytes(a_rows * k if a.dtype == torch.bfloat16 else 0), a.device)
    fn = lib().b200_moe_gemm_loads_only if loads_only else lib().b200_moe_gemm
    _lib.check(
        fn(
            quant, _vp(a), _code(a, "a"), a_rows, k, _vp(packed), _vp(scales), _vp(global_scale),
            num_experts, n, gated_mode, _vp(sorted_token_ids), _vp(expert_ids), groups,
            _vp(num_tokens_post_pad), block_size, top_k, num_routes, _vp(topk_weights),
            int(mul_topk_weights), _vp(c), _code(c, "c"), c.shape[-1], _vp(ws), ws.numel(),
            _stream(a.device),
        )
    )
    return c


def moe_layer_workspace_bytes(tokens: int, hidden: int, inter: int, num_experts: int,
                              top_k: int, block_size: int) -> int:
    return int(lib().b200_moe_layer_workspace_bytes(tokens, hidden, inter, num_experts, top_k, block_size))


def moe_layer_forward(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, *,
                      quant: int, num_experts: int, inter: int, w13: torch.Tensor,
                      w2: torch.Tensor, w13_scales: torch.Tensor | None = None,
                      w2_scales: torch.Tensor | None = None,
                      w13_global: torch.Tensor | None = None,
                      w2_global: torch.Tensor | None = None, block_size: int = 16,
                      routed_scaling_factor: float = 1.0, shared_out: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """align -> gate_up(+SiLU*up) -> down(x weight) -> combine, one library call."""
    _contig(x, "x")
    _contig(topk_ids, "topk_ids")
    _contig(topk_weights, "topk_weights")
    if topk_ids.dtype != torch.int32:
        raise TypeError(f"topk_ids must be int32, got {topk_ids.dtype}")
    if topk_weights.dtype != torch.float32:
        raise TypeError(f"topk_weights must be float32, got {topk_weights.dtype}")
    tokens, hidden = (int(d) for d in x.shape)
    top_k = int(topk_ids.shape[1])
    if out is None:
        out = torch.empty(tokens, hidden, dtype=x.dtype, device=x.device)
    if shared_out is not None:
        _contig(shared_out, "shared_out")
    ws = workspace(
        moe_layer_workspace_bytes(tokens, hidden, inter, num_experts, top_k, block_size), x.device
    )
    _lib.check(
        lib().b200_moe_layer_forward(
            quant, _vp(x), _code(x, "x"), tokens, hidden, inter, _vp(topk_ids), _vp(topk_weights),
            top_k, num_experts, _vp(w13), _vp(w13_scales), _vp(w13_global), _vp(w2),
            _vp(w2_scales), _vp(w2_global), block_size, float(routed_scaling_factor),
            _vp(shared_out), _code(shared_out, "shared_out") if shared_out is not None else 0,
            _vp(out), _code(out, "out"), _vp(ws), ws.numel(), _stream(x.device),
        )
    )
    return out


def moe_layer_forward_fused_shared(x: torch.Tensor, topk_ids: torch.Tensor,
                                   topk_weights: torch.Tensor, *, quant: int, num_experts: int,
                                   inter: int, w13: torch.Tensor, w2: torch.Tensor,
                                   w13_scales: torch.Tensor | None = None,
                                   w2_scales: torch.Tensor | None = None, block_size: int = 16,
                                   routed_scaling_factor: float = 1.0,
                                   shared_route_weight: float | None = None,
                                   out: torch.Tensor | None = None):
    """The layer with the shared expert as the banks' last expert (index
    ``num_experts``, the routed count): one more route per token, appended
    inside the call. Returns (out, extended ids, extended weights), the
    routes [T, top_k + 1] the layer ran on."""
    _contig(x, "x")
    _contig(topk_ids, "topk_ids")
    _contig(topk_weights, "topk_weights")
    if topk_ids.dtype != torch.int32:
        raise TypeError(f"topk_ids must be int32, got {topk_ids.dtype}")
    if topk_weights.dtype != torch.float32:
        raise TypeError(f"topk_weights must be float32, got {topk_weights.dtype}")
    tokens, hidden = (int(d) for d in x.shape)
    top_k = int(topk_ids.shape[1])
    if shared_route_weight is None:
        shared_route_weight = 1.0 / routed_scaling_factor
    ids = torch.empty(tokens, top_k + 1, dtype=torch.int32, device=x.device)
    w = torch.empty(tokens, top_k + 1, dtype=torch.float32, device=x.device)
    if out is None:
        out = torch.empty(tokens, hidden, dtype=x.dtype, device=x.device)
    ws = workspace(
        moe_layer_workspace_bytes(tokens, hidden, inter, num_experts + 1, top_k + 1, block_size),
        x.device,
    )
    _lib.check(
        lib().b200_moe_layer_forward_fused_shared(
            quant, _vp(x), _code(x, "x"), tokens, hidden, inter, _vp(topk_ids), _vp(topk_weights),
            top_k, num_experts, float(shared_route_weight), _vp(ids), _vp(w), _vp(w13),
            _vp(w13_scales), None, _vp(w2), _vp(w2_scales), None, block_size,
            float(routed_scaling_factor), _vp(out), _code(out, "out"), _vp(ws), ws.numel(),
            _stream(x.device),
        )
    )
    return out, ids, w


def moe_layer_forward_logits(x: torch.Tensor, router_logits: torch.Tensor, top_k: int, *,
                             quant: int, num_experts: int, inter: int, w13: torch.Tensor,
                             w2: torch.Tensor, w13_scales=None, w2_scales=None, w13_global=None,
                             w2_global=None, block_size: int = 16,
                             routed_scaling_factor: float = 1.0,
                             shared_out: torch.Tensor | None = None,
                             scoring: int = _lib.SCORING_SOFTMAX, renormalize: bool = True,
                             correction_bias: torch.Tensor | None = None,
                             out: torch.Tensor | None = None):
    """Router top-k + layer in one library call: (out, topk_ids, topk_weights)."""
    _contig(x, "x")
    _contig(router_logits, "router_logits")
    try:
        lcode = _LOGIT_CODE[router_logits.dtype]
    except KeyError:
        raise TypeError(f"router_logits must be bf16, f16 or f32, got {router_logits.dtype}") from None
    tokens, hidden = (int(d) for d in x.shape)
    if correction_bias is not None:
        _contig(correction_bias, "correction_bias")
    ids = torch.empty(tokens, top_k, dtype=torch.int32, device=x.device)
    w = torch.empty(tokens, top_k, dtype=torch.float32, device=x.device)
    if out is None:
        out = torch.empty(tokens, hidden, dtype=x.dtype, device=x.device)
    if shared_out is not None:
        _contig(shared_out, "shared_out")
    ws = workspace(
        moe_layer_workspace_bytes(tokens, hidden, inter, num_experts, top_k, block_size), x.device
    )
    _lib.check(
        lib().b200_moe_layer_forward_logits(
            quant, _vp(x), _code(x, "x"), tokens, hidden, inter, _vp(router_logits), lcode,
            scoring, int(renormalize), _vp(correction_bias), top_k, num_experts, _vp(ids), _vp(w),
            _vp(w13), _vp(w13_scales), _vp(w13_global), _vp(w2), _vp(w2_scales), _vp(w2_global),
            block_size, float(routed_scaling_factor), _vp(shared_out),
            _code(shared_out, "shared_out") if shared_out is not None else 0, _vp(out),
            _code(out, "out"), _vp(ws), ws.numel(), _stream(x.device),
        )
    )
    return out, ids, w


# ------------------------------------------------------ expert parallelism
# Peer-memory exchange (b200_ep_*): see ep.PeerExchange for the set-up of the
# per-rank regions and their mapping into every peer.
def ep_region_bytes(world: int, max_tokens: int, top_k: int, hidden: int) -> int:
    n = int(lib().b200_ep_region_bytes(world, max_tokens, top_k, hidden))
    if n < 0:
        raise ValueError("bad expert-parallel region shape")
    return n


def ep_region_layout(world: int, max_tokens: int, top_k: int, hidden: int) -> dict:
    """Byte offsets of a region's arrays (see b200_ep_region_layout)."""
    arr = (ctypes.c_int64 * 7)()
    _lib.check(lib().b200_ep_region_layout(world, max_tokens, top_k, hidden, arr))
    keys = ("ids", "weights", "orig", "rows", "recv", "comb", "total")
    return dict(zip(keys, (int(v) for v in arr)))


def aligned_zeros(nbytes: int, device: torch.device) -> torch.Tensor:
    """Zero-filled uint8 buffer of ``nbytes`` whose base is 256-byte aligned."""
    raw = torch.zeros(nbytes + 256, dtype=torch.uint8, device=device)
    offset = (-raw.data_ptr()) % 256
    return raw[offset : offset + nbytes]


def ipc_get_handle(t: torch.Tensor) -> tuple[bytes, int]:
    """(64-byte CUDA IPC handle of t's allocation, t's offset inside it)."""
    _cuda(t, "buffer")
    handle = ctypes.create_string_buffer(64)
    offset = ctypes.c_int64(0)
    _lib.check(lib().b200_ipc_get_handle(_vp(t), handle, ctypes.byref(offset)))
    return handle.raw, int(offset.value)


def ipc_open_handle(handle: bytes, offset: int) -> int:
    """Maps a peer's allocation; returns the device address of its buffer."""
    if len(handle) != 64:
        raise ValueError("an IPC handle is 64 bytes")
    ptr = ctypes.c_void_p(0)
    _lib.check(lib().b200_ipc_open_handle(ctypes.create_string_buffer(handle, 64), int(offset),
                                          ctypes.byref(ptr)))
    return int(ptr.value)


def ipc_close_handle(address: int, offset: int) -> None:
    _lib.check(lib().b200_ipc_close_handle(ctypes.c_void_p(address), int(offset)))


def _peers_arg(peers: torch.Tensor, world: int):
    _contig(peers, "peer_regions")
    if peers.dtype != torch.int64 or peers.numel() != world:
        raise ValueError(f"peer_regions must be int64[{world}] on the device")
    return _vp(peers)


def ep_dispatch(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, *,
                num_experts: int, rank: int, world: int, peers: torch.Tensor,
                region: torch.Tensor, max_tokens: int, shared_expert: bool = False) -> None:
    """Source side: this rank's routes (rows + routing) into their owners' regions."""
    _contig(x, "x")
    _contig(topk_ids, "topk_ids")
    _contig(topk_weights, "topk_weights")
    _contig(region, "region")
    if topk_ids.dtype != torch.int32 or topk_weights.dtype != torch.float32:
        raise TypeError("topk_ids must be int32 and topk_weights float32")
    tokens, hidden = (int(d) for d in x.shape)
    _lib.check(
        lib().b200_ep_dispatch(
            _vp(x), _code(x, "x"), tokens, hidden, _vp(topk_ids), _vp(topk_weights),
            int(topk_ids.shape[1]), num_experts, int(shared_expert), rank, world,
            _peers_arg(peers, world), _vp(region), max_tokens, _stream(x.device),
        )
    )


def ep_expert_workspace_bytes(world: int, max_tokens: int, top_k: int, hidden: int, inter: int,
                              local_experts: int, block_size: int) -> int:
    return int(lib().b200_ep_expert_workspace_bytes(world, max_tokens, top_k, hidden, inter,
                                                    local_experts, block_size))


def ep_expert_forward(*, quant: int, hidden: int, inter: int, local_experts: int,
                      w13: torch.Tensor, w2: torch.Tensor, w13_scales=None, w2_scales=None,
                      w13_global=None, w2_global=None, block_size: int, rank: int, world: int,
                      peers: torch.Tensor, region: torch.Tensor, max_tokens: int,
                      top_k: int) -> None:
    """Owner side: wait for every source, run this rank's experts on what
    arrived, store each weighted row into its source's region."""
    _contig(region, "region")
    ws = workspace(
        ep_expert_workspace_bytes(world, max_tokens, top_k, hidden, inter, local_experts,
                                  block_size),
        region.device,
    )
    _lib.check(
        lib().b200_ep_expert_forward(
            quant, hidden, inter, local_experts, _vp(w13), _vp(w13_scales), _vp(w13_global),
            _vp(w2), _vp(w2_scales), _vp(w2_global), block_size, rank, world,
            _peers_arg(peers, world), _vp(region), max_tokens, top_k, _vp(ws), ws.numel(),
            _stream(region.device),
        )
    )


def ep_combine(topk_ids: torch.Tensor, *, hidden: int, num_experts: int, world: int,
               region: torch.Tensor, max_tokens: int, routed_scaling_factor: float = 1.0,
               shared_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Source side: wait for every owner, sum each token's returned rows."""
    _contig(topk_ids, "topk_ids")
    _contig(region, "region")
    tokens, top_k = (int(d) for d in topk_ids.shape)
    if out is None:
        out = torch.empty(tokens, hidden, dtype=out_dtype, device=topk_ids.device)
    _contig(out, "out")
    if shared_out is not None:
        _contig(shared_out, "shared_out")
    _lib.check(
        lib().b200_ep_combine(
            tokens, hidden, _vp(topk_ids), top_k, num_experts, float(routed_scaling_factor),
            _vp(shared_out), _code(shared_out, "shared_out") if shared_out is not None else 0,
            _vp(out), _code(out, "out"), world, _vp(region), max_tokens, _stream(out.device),
        )
    )
    return out


def region_status(region: torch.Tensor, reset: bool = True) -> int:
    """Error bits of an expert-parallel region (8 = a wait on a peer timed out). Synchronizes."""
    bits = ctypes.c_int32(0)
    _lib.check(lib().b200_workspace_status(_vp(region), ctypes.byref(bits), int(reset),
                                           _stream(region.device)))
    return int(bits.value)


# ------------------------------------------- W8A8 block FP8 (opt-in path)
# FP8 x FP8 on the tensor cores; the activations are quantized per (row,
# 128-K group), so results differ from the W8A16 ops above. Weights are the
# checkpoint's row-major e4m3 [E, N, K] with fp32 scales [E, N/128, K/128].
def w8a8_workspace_bytes(slots: int, k: int) -> int:
    n = int(lib().b200_w8a8_workspace_bytes(int(slots), int(k)))
    if n < 0:
        raise ValueError(f"bad W8A8 workspace shape slots={slots} k={k}")
    return n


def fp8_act_quant(x: torch.Tensor, scales_ld: int | None = None):
    """(q e4m3 [rows, K], scales fp32 [K/128, scales_ld]) of bf16/f16 ``x``:
    scale = max(amax / 448, 1e-8) per (row, 128-K group)."""
    _contig(x, "x")
    rows, k = (int(d) for d in x.shape)
    ld = rows if scales_ld is None else int(scales_ld)
    q = torch.empty(rows, k, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty(k // 128, ld, dtype=torch.float32, device=x.device)
    _lib.check(lib().b200_fp8_act_quant(_vp(x), _code(x, "x"), rows, k, _vp(q), _vp(s), ld,
                                        _stream(x.device)))
    return q, s


def _w8_weights(w: torch.Tensor, w_scales: torch.Tensor):
    _contig(w, "weight")
    _contig(w_scales, "weight scales")
    if w.dtype != torch.float8_e4m3fn:
        raise TypeError(f"W8A8 weights must be float8_e4m3fn, got {w.dtype}")
    if w_scales.dtype != torch.float32:
        raise TypeError(f"W8A8 weight scales must be float32, got {w_scales.dtype}")


def w8a8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *,
                gated_mode: int = _lib.GATED_NONE, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``y = W8A8(x, W)`` with W row-major e4m3 ``[N, K]`` and scales ``[N/128, K/128]``."""
    _contig(x, "x")
    _w8_weights(w, w_scales)
    x2 = x.reshape(-1, x.shape[-1])
    m, k = (int(d) for d in x2.shape)
    n = int(w.shape[-2])
    cols = n // 2 if gated_mode == _lib.GATED_FUSED else n
    if out is None:
        out = torch.empty(m, cols, dtype=out_dtype or x.dtype, device=x.device)
    ws = workspace(w8a8_workspace_bytes(m, k), x.device)
    _lib.check(
        lib().b200_w8a8_linear(_vp(x2), _code(x2, "x"), m, k, _vp(w), _vp(w_scales), n, gated_mode,
                               _vp(out), _code(out, "out"), _vp(ws), ws.numel(), _stream(x.device))
    )
    return out.reshape(*x.shape[:-1], cols)


def w8a8_moe_gemm(a: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *, num_experts: int,
                  sorted_token_ids: torch.Tensor, expert_ids: torch.Tensor,
                  num_tokens_post_pad: torch.Tensor, block_size: int, top_k: int, num_routes: int,
                  c: torch.Tensor, topk_weights: torch.Tensor | None = None,
                  mul_topk_weights: bool = False, gated_mode: int = _lib.GATED_NONE) -> torch.Tensor:
    """Grouped W8A8 expert GEMM with ``moe_wna16_marlin_gemm`` routing semantics;
    ``w`` e4m3 ``[E, N, K]`` row-major, ``w_scales`` ``[E, N/128, K/128]``."""
    _contig(a, "a")
    _contig(c, "c")
    _w8_weights(w, w_scales)
    a_rows, k = (int(d) for d in a.reshape(-1, a.shape[-1]).shape)
    n = int(w.shape[-2])
    if topk_weights is not None:
        topk_weights = topk_weights.reshape(-1).float().contiguous()
    if c.shape[0] < num_routes:
        raise ValueError(f"c has {c.shape[0]} rows, the routes need {num_routes}")
    if mul_topk_weights and (topk_weights is None or topk_weights.numel() < num_routes):
        raise ValueError("mul_topk_weights needs one topk weight per route")
    groups = min(expert_ids.numel(), sorted_token_ids.numel() // block_size)
    ws = workspace(w8a8_workspace_bytes(groups * block_size, k), a.device)
    _lib.check(
        lib().b200_w8a8_moe_gemm(
            _vp(a), _code(a, "a"), a_rows, k, _vp(w), _vp(w_scales), num_experts, n, gated_mode,
            _vp(sorted_token_ids), _vp(expert_ids), groups, _vp(num_tokens_post_pad), block_size,
            top_k, num_routes, _vp(topk_weights), int(mul_topk_weights), _vp(c), _code(c, "c"),
            c.shape[-1], _vp(ws), ws.numel(), _stream(a.device),
        )
    )
    return c


def w8a8_scales_ld(rows: int) -> int:
    """Leading dimension of activation scales that :func:`w8a8_linear_quantized` takes."""
    return (rows + 127) // 128 * 128


def w8a8_linear_quantized(q: torch.Tensor, scales: torch.Tensor, w: torch.Tensor,
                          w_scales: torch.Tensor, *, gated_mode: int = _lib.GATED_NONE,
                          out: torch.Tensor | None = None,
                          out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`w8a8_linear` on activations that are already quantized: ``q`` e4m3
    ``[M, K]`` and ``scales`` fp32 ``[K/128, >= w8a8_scales_ld(M)]``, as
    :func:`fp8_act_quant` or :func:`add_rms_norm_fp8` return them."""
    _contig(q, "q")
    _contig(scales, "scales")
    _w8_weights(w, w_scales)
    if q.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32:
        raise TypeError(f"q must be float8_e4m3fn and scales float32, got {q.dtype}, {scales.dtype}")
    if q.dim() != 2 or scales.dim() != 2:
        raise ValueError(f"q must be [M, K] and scales [K/128, ld], got {tuple(q.shape)}, "
                         f"{tuple(scales.shape)}")
    m, k = (int(d) for d in q.shape)
    if w.shape[-1] != k or scales.shape[0] != k // 128:
        raise ValueError(f"K differs: q {k}, weight {w.shape[-1]}, scales {scales.shape[0]} groups")
    n = int(w.shape[-2])
    if w.numel() != n * k or w_scales.numel() != n // 128 * (k // 128):
        raise ValueError(f"weight must be [N, K] with scales [N/128, K/128], got {tuple(w.shape)}, "
                         f"{tuple(w_scales.shape)}")
    if any(t.device != q.device for t in (scales, w, w_scales)):
        raise ValueError("w8a8_linear_quantized: the operands are on different devices")
    cols = n // 2 if gated_mode == _lib.GATED_FUSED else n
    if out is None:
        out = torch.empty(m, cols, dtype=out_dtype, device=q.device)
    elif out.shape != (m, cols) or not out.is_contiguous() or out.device != q.device:
        raise ValueError(f"out must be a contiguous [{m}, {cols}] on {q.device}, got "
                         f"{tuple(out.shape)} on {out.device}")
    ws = workspace(gemm_workspace_bytes(0), q.device)
    _lib.check(
        lib().b200_w8a8_linear_quantized(
            _vp(q), _vp(scales), scales.shape[1], m, k, _vp(w), _vp(w_scales), n, gated_mode,
            _vp(out), _code(out, "out"), _vp(ws), ws.numel(), _stream(q.device))
    )
    return out


# --------------------------------------------------- 8-bit integer linear
def _int8_weights(w: torch.Tensor, w_scales: torch.Tensor, k: int) -> int:
    if w.dtype != torch.int8 or w_scales.dtype != torch.float32:
        raise TypeError(f"the weight must be int8 and its scales float32, got {w.dtype}, "
                        f"{w_scales.dtype}")
    if w.dim() != 2 or w.shape[1] != k or w_scales.shape != w.shape[:1]:
        raise ValueError(f"the weight must be [N, {k}] with scales [N], got {tuple(w.shape)}, "
                         f"{tuple(w_scales.shape)}")
    if not w.is_contiguous() or not w_scales.is_contiguous():
        raise ValueError("the weight and its scales must be contiguous")
    return int(w.shape[0])


def _int8_rows(t: torch.Tensor, what: str) -> None:
    if t.dim() != 2 or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous [M, K], got {tuple(t.shape)} strides {t.stride()}")


def _int8_out(out, m, n, dtype, device):
    if out is None:
        return torch.empty(m, n, dtype=dtype, device=device)
    if out.shape != (m, n) or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous [{m}, {n}], got {tuple(out.shape)} "
                         f"strides {out.stride()}")
    return out


def int8_act_quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token quantization of ``x`` ``[M, K]`` (bf16 or f16): ``scale = max|x| /
    127``, int8 codes ``rint(x / scale)``. A token with an infinity or NaN has a NaN
    scale. Returns (codes ``[M, K]``, fp32 scales ``[M]``)."""
    index = _on_device("int8_act_quant", x)
    _int8_rows(x, "x")
    m, k = x.shape
    code = _code(x, "x")
    q = torch.empty(m, k, dtype=torch.int8, device=x.device)
    scales = torch.empty(m, dtype=torch.float32, device=x.device)
    _lib.check(lib().b200_int8_act_quant(x.data_ptr(), code, m, k, q.data_ptr(), scales.data_ptr(),
                                         _raw_stream(index)))
    return q, scales


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *,
                out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``y = x W^T`` with 8-bit integer products: ``x`` ``[..., K]`` (bf16 or f16) is
    quantized per token as :func:`int8_act_quant` does, ``w`` int8 ``[N, K]`` has an
    fp32 scale per output channel ``[N]``. K a multiple of 16; any N. ``out``
    ``[M, N]`` and ``out_dtype``: bf16 or f16, by default ``x``'s type."""
    index = _on_device("int8_linear", x, w, w_scales, out)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    _int8_rows(x2, "x")
    m, k = x2.shape
    n = _int8_weights(w, w_scales, k)
    code = _code(x2, "x")
    out = _int8_out(out, m, n, out_dtype or x.dtype, x.device)
    # the codes and their scales, in one allocation
    buf = torch.empty(m * k + 4 * m, dtype=torch.int8, device=x.device)
    _lib.check(lib().b200_int8_linear(
        x2.data_ptr(), code, m, k, w.data_ptr(), w_scales.data_ptr(), n, buf.data_ptr(),
        buf.data_ptr() + m * k, out.data_ptr(), _code(out, "out"), _raw_stream(index)))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], n)


def int8_linear_quantized(q: torch.Tensor, scales: torch.Tensor, w: torch.Tensor,
                          w_scales: torch.Tensor, *, out: torch.Tensor | None = None,
                          out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`int8_linear` on activations that are already quantized: ``q`` int8
    ``[M, K]`` and fp32 ``scales`` ``[M]``, as :func:`int8_act_quant` returns them."""
    index = _on_device("int8_linear_quantized", q, scales, w, w_scales, out)
    _int8_rows(q, "q")
    m, k = q.shape
    if q.dtype != torch.int8 or scales.dtype != torch.float32:
        raise TypeError(f"q must be int8 and scales float32, got {q.dtype}, {scales.dtype}")
    if scales.shape != (m,) or not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous [{m}], got {tuple(scales.shape)}")
    n = _int8_weights(w, w_scales, k)
    out = _int8_out(out, m, n, out_dtype, q.device)
    _lib.check(lib().b200_int8_linear_quantized(
        q.data_ptr(), scales.data_ptr(), m, k, w.data_ptr(), w_scales.data_ptr(), n, out.data_ptr(),
        _code(out, "out"), _raw_stream(index)))
    return out


# ------------------------------------------- norm, key/value cache, attention
# Decode calls these several times a layer on microseconds of GPU work, so the
# wrappers keep their own host time low: plain integers instead of ctypes
# objects, and the current stream and device by their raw handles.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _on_device(what: str, *tensors: torch.Tensor | None) -> int:
    """The index of the one CUDA device all tensors are on; it must be the
    current one, whose context the library launches in."""
    index = _current_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            if not t.is_cuda:
                raise ValueError(f"{what}: operands must be CUDA tensors")
            raise ValueError(f"{what}: an operand is on {t.device}, the current device is "
                             f"cuda:{index}")
    return index


def _norm(x, weight, eps, residual, weight_bias, residual_out, y, q, scales, scales_ld, like):
    index = _on_device("add_rms_norm", x, weight, residual, residual_out, y)
    dtype, shape = x.dtype, x.shape
    code = _DTYPE_CODE.get(dtype)
    wcode = _LOGIT_CODE.get(weight.dtype)
    if code is None or wcode is None:
        raise TypeError(f"x must be bf16 or f16 and weight bf16, f16 or f32, got {dtype}, "
                        f"{weight.dtype}")
    rows, hidden = shape
    if weight.shape != (hidden,) or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous [{hidden}], got {tuple(weight.shape)}")
    ptrs = []  # residual, residual_out, y: address and leading dimension
    for t in (residual, residual_out, y):
        if t is None:
            ptrs += (None, 0)
            continue
        ld, one = t.stride()
        if t.shape != shape or t.dtype != dtype or one != 1:
            raise ValueError(f"{like} must be {tuple(shape)} {dtype} rows, got "
                             f"{tuple(t.shape)} {t.dtype}")
        ptrs += (t.data_ptr(), ld)
    status = lib().b200_add_rms_norm(
        x.data_ptr(), code, x.stride(0), rows, hidden, ptrs[0], ptrs[1], weight.data_ptr(), wcode,
        weight_bias, eps, ptrs[2], ptrs[3], ptrs[4], ptrs[5],
        None if q is None else q.data_ptr(), None if scales is None else scales.data_ptr(),
        scales_ld, _raw_stream(index))
    if status:
        _lib.check(status)


def _norm_rows(x: torch.Tensor) -> None:
    if x.dim() != 2 or x.stride(-1) != 1:
        raise ValueError("x must be [rows, hidden] with contiguous rows")


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                 residual: torch.Tensor | None = None, weight_bias: float = 0.0,
                 out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None):
    """``(y, h)``: ``h = x + residual`` (``None`` without a residual) and ``y = h *
    rsqrt(mean(h^2) + eps) * (weight + weight_bias)``, both in ``x``'s type.

    ``x``, ``residual`` and the outputs are ``[rows, hidden]`` with contiguous
    rows; ``out`` and ``residual_out`` may be ``x`` or ``residual`` (in place)."""
    _norm_rows(x)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if residual is not None and residual_out is None:
        residual_out = torch.empty_like(x, memory_format=torch.contiguous_format)
    _norm(x, weight, eps, residual, weight_bias, residual_out, out, None, None, 0,
          "residual, residual_out and out")
    return out, residual_out


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                     residual: torch.Tensor | None = None, weight_bias: float = 0.0,
                     residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     scales_ld: int | None = None):
    """``(q, scales, h)``: :func:`add_rms_norm` with its output quantized as
    :func:`fp8_act_quant` does (e4m3 ``[rows, hidden]``, fp32 scales ``[hidden /
    128, scales_ld]``, default ``scales_ld = rows``; pass ``w8a8_scales_ld(rows)``
    for :func:`w8a8_linear_quantized`). ``out``: also store the 16-bit output."""
    _norm_rows(x)
    rows, hidden = x.shape
    ld = rows if scales_ld is None else int(scales_ld)
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    scales = x.new_empty((hidden // 128, ld), dtype=torch.float32)
    if residual is not None and residual_out is None:
        residual_out = torch.empty_like(x, memory_format=torch.contiguous_format)
    _norm(x, weight, eps, residual, weight_bias, residual_out, out, q, scales, ld,
          "residual, residual_out and out")
    return q, scales, residual_out


def _vectors(t: torch.Tensor, cache, what: str) -> None:
    if t.dim() != 3 or t.shape[1] != cache.kv_heads or t.shape[2] != cache.head_dim \
            or t.stride(2) != 1:
        raise ValueError(f"{what} must be [tokens, {cache.kv_heads}, {cache.head_dim}] with "
                         f"contiguous vectors, got {tuple(t.shape)} strides {t.stride()}")


def _slots(slots: torch.Tensor, tokens: int | None = None) -> None:
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int64 [tokens]")
    if tokens is not None and slots.shape[0] != tokens:
        raise ValueError(f"{slots.shape[0]} slots for {tokens} tokens")


def kv_cache_write(cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes ``k`` and ``v`` ``[tokens, kv_heads, head_dim]`` (any strides over
    tokens and heads) into their slots (int64 ``page * page_size + offset``;
    negative: skipped), quantized when the cache is e4m3."""
    index = _on_device("kv_cache_write", k, v, slots, cache.k)
    _vectors(k, cache, "k")
    _vectors(v, cache, "v")
    _slots(slots, k.shape[0])
    code = _DTYPE_CODE.get(k.dtype)
    if code is None or v.dtype != k.dtype or v.shape[0] != k.shape[0]:
        raise TypeError(f"k and v must be bf16 or f16 alike, got {k.dtype} {tuple(k.shape)}, "
                        f"{v.dtype} {tuple(v.shape)}")
    _lib.check(
        lib().b200_kv_cache_write(cache.desc, k.data_ptr(), v.data_ptr(), code, k.stride(0),
                                  k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(),
                                  k.shape[0], _raw_stream(index))
    )


def kv_cache_read(cache, slots: torch.Tensor, dtype: torch.dtype | None = None):
    """``(k, v)`` ``[tokens, kv_heads, head_dim]`` of the given slots as values
    (zeros for slots outside the cache). ``dtype``: bf16 or f16, by default the
    cache's own, bf16 for an e4m3 cache."""
    index = _on_device("kv_cache_read", slots, cache.k)
    _slots(slots)
    if dtype is None:
        dtype = torch.bfloat16 if cache.k_scale is not None else cache.k.dtype
    code = _DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"dtype must be bf16 or f16, got {dtype}")
    n = slots.shape[0]
    k = torch.empty(n, cache.kv_heads, cache.head_dim, dtype=dtype, device=slots.device)
    v = torch.empty_like(k)
    _lib.check(
        lib().b200_kv_cache_read(cache.desc, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), code,
                                 cache.kv_heads * cache.head_dim, cache.head_dim,
                                 _raw_stream(index))
    )
    return k, v


# Attention keeps one workspace per (device, stream): calls on two streams may
# overlap, and its arrival counters and partial sums must not.
_ATTN_WORKSPACES: dict[tuple[int, int], torch.Tensor] = {}
_ATTN_BYTES: dict[tuple[int, int, int], int] = {}
_PREFIX_BYTES: dict[tuple[int, int, int, int, int], int] = {}
_SCORES_BYTES: dict[tuple[int, int, int], int] = {}
# Workspaces that a larger one has replaced, kept because a captured graph may still
# use them. Each is at most half of the one after it, so a stream's together are
# below its present one. (Without shared prefixes nearly all of a workspace is its
# partial results, a constant: 20 to 40 MB by head_dim, and 16 bytes a token. Shared
# prefixes add 8 bytes a query element, scores over an e4m3 cache 3: a chunk of 16384
# tokens with 64 heads of 128 takes 1.1 GB and 0.4 GB, which stay.)
_ATTN_OUTGROWN: list[torch.Tensor] = []
_ATTN_MIN_TOKENS, _ATTN_MIN_SEQS = 16384, 4096


def paged_attention_workspace_bytes(head_dim: int, q_tokens: int, seqs: int) -> int:
    n = int(lib().b200_paged_attention_workspace_bytes(head_dim, q_tokens, seqs))
    if n < 0:
        raise ValueError(f"no attention kernel for head_dim {head_dim}")
    return n


def _rounded(q_tokens: int, seqs: int) -> tuple[int, int]:
    # Sizes are asked for rounded up: few distinct ones, and no growth up to the
    # minimum, which costs a hundredth.
    return (max(_ATTN_MIN_TOKENS, 1 << max(0, q_tokens - 1).bit_length()),
            max(_ATTN_MIN_SEQS, 1 << max(0, seqs - 1).bit_length()))


def _attn_workspace(index: int, stream: int, head_dim: int, q_tokens: int, seqs: int):
    key = (head_dim, *_rounded(q_tokens, seqs))
    nbytes = _ATTN_BYTES.get(key)
    if nbytes is None:
        nbytes = _ATTN_BYTES[key] = paged_attention_workspace_bytes(*key)
    return _attn_workspace_of(index, stream, nbytes)


def _attn_workspace_of(index: int, stream: int, nbytes: int):
    ws = _ATTN_WORKSPACES.get((index, stream))
    if ws is not None and ws.numel() >= nbytes:
        return ws
    if torch.cuda.is_current_stream_capturing():
        # A capture runs on a stream of its own: this call's workspace comes
        # from the graph's pool, and each replay clears the part that counts
        # arrivals. reserve_attention_workspace() on the capturing stream, or
        # the workspace argument, saves the clearing.
        ws = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
        ws[:8192].zero_()
        return ws
    with _WS_LOCK:
        old = _ATTN_WORKSPACES.get((index, stream))
        if old is not None and old.numel() >= nbytes:
            return old  # another thread's, meanwhile
        if old is not None:
            nbytes = max(nbytes, 2 * old.numel())
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
        if old is not None:
            _ATTN_OUTGROWN.append(old)
        _ATTN_WORKSPACES[(index, stream)] = ws
    return ws


def reserve_attention_workspace(head_dim: int, q_tokens: int, seqs: int,
                                device: torch.device | None = None) -> torch.Tensor:
    """The current stream's attention workspace, for calls of up to these sizes.

    Calls captured on this stream then use it instead of clearing one of their own
    in each replay. They share its counters and partial results with every other
    call on it: graphs captured so, and calls on this stream, must not run at the
    same time (replay them on one stream, or join the streams by events)."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    return _attn_workspace(index, _raw_stream(index), head_dim, q_tokens, seqs)


def attention_status(device: torch.device | None = None, reset: bool = True) -> int:
    """Error bits of a device's norm, attention, integer linear, score and eviction
    calls, those replayed from graphs included (0 = none, 1 = a wait gave up, 16 = a
    page number outside the cache, 32 = a chunk met a scale byte outside 103 .. 134).
    Synchronizes the device."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    torch.cuda.synchronize(index)
    bits = ctypes.c_int32(0)
    with torch.cuda.device(index):
        _lib.check(lib().b200_device_status(ctypes.byref(bits), int(reset), _raw_stream(index)))
    return int(bits.value)


def _attention_args(q, cache, page_table, kv_lens, q_starts, out):
    """(dtype code, tokens, heads, head_dim, sequences, out) of an attention call."""
    dtype = q.dtype
    code = _DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"q must be bf16 or f16, got {dtype}")
    if q.dim() != 3 or q.shape[2] != cache.head_dim or q.stride(2) != 1:
        raise ValueError(f"q must be [tokens, heads, {cache.head_dim}] with contiguous vectors, "
                         f"got {tuple(q.shape)} strides {q.stride()}")
    tokens, heads, dim = q.shape
    seqs = kv_lens.shape[0]
    _tables((page_table, "page_table"), (kv_lens, "kv_lens"), (q_starts, "q_starts"))
    if q_starts.shape[0] != seqs + 1 or page_table.dim() != 2 or page_table.shape[0] != seqs:
        raise ValueError(f"{seqs} sequences need q_starts [{seqs + 1}] and page_table [{seqs}, "
                         f"pages], got {tuple(q_starts.shape)}, {tuple(page_table.shape)}")
    if out is None:
        out = torch.empty(tokens, heads, dim, dtype=dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != dtype or out.stride(2) != 1:
        raise ValueError(f"out must be {tuple(q.shape)} {dtype}, got {tuple(out.shape)} {out.dtype}")
    return code, tokens, heads, dim, seqs, out


def _tables(*named) -> None:
    for t, what in named:
        if t.dtype != torch.int32 or t.stride(-1) != 1:
            raise ValueError(f"{what} must be int32 with contiguous rows, got {t.dtype}")


def _own_workspace(ws: torch.Tensor) -> torch.Tensor:
    if ws.dtype != torch.uint8 or not ws.is_contiguous():
        raise TypeError(f"the workspace must be contiguous uint8, got {ws.dtype}")
    return ws


def paged_attention(q: torch.Tensor, cache, page_table: torch.Tensor, kv_lens: torch.Tensor,
                    q_starts: torch.Tensor, max_q_len: int, *, scale: float | None = None,
                    causal: bool = True, window: int = 0, out: torch.Tensor | None = None,
                    return_lse: bool = False, workspace: torch.Tensor | None = None):
    """Attention of each sequence's new tokens over its cached ones.

    ``q`` ``[tokens, q_heads, head_dim]`` holds the new tokens of all sequences
    (sequence s: rows ``q_starts[s] : q_starts[s + 1]``, at most ``max_q_len``),
    which are the last of its ``kv_lens[s]`` tokens in ``cache`` (a
    :class:`~.kv_cache.PagedKVCache`; write them first), on the pages
    ``page_table[s]`` (int32 ``[seqs, pages]``). ``causal`` masks by position,
    ``window`` (causal only; 0: none) keeps the last ``window`` positions. Rows
    that see nothing give zeros and ``-inf``. ``scale`` defaults to
    ``head_dim ** -0.5``. Returns ``out``, or ``(out, lse)`` with the fp32
    ``[tokens, q_heads]`` log-sum-exp. A few new tokens (``max_q_len * q_heads /
    kv_heads`` up to 8 or 16, by type and head size) stream the cache; larger calls
    run on the tensor cores' kernel."""
    index = _on_device("paged_attention", q, cache.k, page_table, kv_lens, q_starts, out,
                       workspace)
    code, tokens, heads, dim, seqs, out = _attention_args(q, cache, page_table, kv_lens, q_starts,
                                                          out)
    lse = torch.empty(tokens, heads, dtype=torch.float32, device=q.device) if return_lse else None
    stream = _raw_stream(index)
    ws = _own_workspace(workspace) if workspace is not None \
        else _attn_workspace(index, stream, dim, tokens, seqs)
    _lib.check(
        lib().b200_paged_attention(
            cache.desc, q.data_ptr(), code, tokens, heads, q.stride(0), q.stride(1),
            page_table.data_ptr(), page_table.stride(0), page_table.shape[1], kv_lens.data_ptr(),
            q_starts.data_ptr(), seqs, max_q_len, dim ** -0.5 if scale is None else scale,
            causal, window, out.data_ptr(), out.stride(0), out.stride(1),
            None if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(), stream)
    )
    return (out, lse) if return_lse else out


def shared_prefix_attention_workspace_bytes(head_dim: int, q_tokens: int, q_heads: int, seqs: int,
                                            groups: int) -> int:
    n = int(lib().b200_shared_prefix_attention_workspace_bytes(head_dim, q_tokens, q_heads, seqs,
                                                               groups))
    if n < 0:
        raise ValueError(f"no attention kernel for head_dim {head_dim}, {q_heads} heads")
    return n


def _prefix_workspace(index: int, stream: int, head_dim: int, q_tokens: int, q_heads: int,
                      seqs: int, groups: int):
    # (the rows in fp32 are most of it: they are not rounded up far)
    key = (head_dim, -(-q_tokens // 256) * 256, q_heads, _rounded(0, seqs)[1],
           _rounded(0, groups)[1])
    nbytes = _PREFIX_BYTES.get(key)
    if nbytes is None:
        nbytes = _PREFIX_BYTES[key] = shared_prefix_attention_workspace_bytes(*key)
    return _attn_workspace_of(index, stream, nbytes)


def reserve_shared_prefix_workspace(head_dim: int, q_tokens: int, q_heads: int, seqs: int,
                                    groups: int, device: torch.device | None = None) -> torch.Tensor:
    """:func:`reserve_attention_workspace` for :func:`shared_prefix_attention` calls of
    up to these sizes; the same workspace serves both."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    return _prefix_workspace(index, _raw_stream(index), head_dim, q_tokens, q_heads, seqs, groups)


def shared_prefix_attention(q: torch.Tensor, cache, prefix_table: torch.Tensor,
                            prefix_lens: torch.Tensor, group_starts: torch.Tensor,
                            page_table: torch.Tensor, kv_lens: torch.Tensor,
                            q_starts: torch.Tensor, max_q_len: int, *, scale: float | None = None,
                            out: torch.Tensor | None = None, return_lse: bool = False,
                            workspace: torch.Tensor | None = None):
    """:func:`paged_attention` of a batch whose sequences share long prefixes, each
    prefix read once for all of its sequences.

    Group g is the sequences ``group_starts[g] : group_starts[g + 1]`` (int32 ``[groups
    + 1]``, from 0 to the number of sequences); its prefix is the first
    ``prefix_lens[g]`` tokens (0: none) of the pages ``prefix_table[g]`` (int32
    ``[groups, pages]``). ``page_table``, ``kv_lens``, ``q_starts`` and ``max_q_len``
    describe each sequence's own tokens, which come after the prefix and begin on a
    page of their own; its new tokens are the last of them. Every new token sees its
    group's whole prefix and its own tokens causally; the log-sum-exp is over both.

    The workspace holds both passes' rows in fp32, 8 bytes a query element, and stays
    with its stream: with many new tokens, call for a part of the sequences at a time."""
    index = _on_device("shared_prefix_attention", q, cache.k, prefix_table, prefix_lens,
                       group_starts, page_table, kv_lens, q_starts, out, workspace)
    code, tokens, heads, dim, seqs, out = _attention_args(q, cache, page_table, kv_lens, q_starts,
                                                          out)
    _tables((prefix_table, "prefix_table"), (prefix_lens, "prefix_lens"),
            (group_starts, "group_starts"))
    groups = prefix_lens.shape[0]
    if group_starts.shape != (groups + 1,) or prefix_table.dim() != 2 \
            or prefix_table.shape[0] != groups:
        raise ValueError(f"{groups} groups need group_starts [{groups + 1}] and prefix_table "
                         f"[{groups}, pages], got {tuple(group_starts.shape)}, "
                         f"{tuple(prefix_table.shape)}")
    lse = torch.empty(tokens, heads, dtype=torch.float32, device=q.device) if return_lse else None
    stream = _raw_stream(index)
    ws = _own_workspace(workspace) if workspace is not None \
        else _prefix_workspace(index, stream, dim, tokens, heads, seqs, groups)
    _lib.check(
        lib().b200_shared_prefix_attention(
            cache.desc, q.data_ptr(), code, tokens, heads, q.stride(0), q.stride(1),
            prefix_table.data_ptr(), prefix_table.stride(0), prefix_table.shape[1],
            prefix_lens.data_ptr(), group_starts.data_ptr(), groups, page_table.data_ptr(),
            page_table.stride(0), page_table.shape[1], kv_lens.data_ptr(), q_starts.data_ptr(), seqs,
            max_q_len, dim ** -0.5 if scale is None else scale, out.data_ptr(), out.stride(0),
            out.stride(1), None if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(), stream)
    )
    return (out, lse) if return_lse else out


# ------------------------------------------------ weights of cached tokens
def _scores_of(scores: torch.Tensor, cache, what: str = "scores") -> None:
    if scores.dtype != torch.float32:
        raise TypeError(f"{what} must be float32, got {scores.dtype}")
    if scores.shape != cache.k.shape[:3]:
        raise ValueError(f"{what} must be {tuple(cache.k.shape[:3])} (pages, page size, heads), got "
                         f"{tuple(scores.shape)}")


def kv_cache_scores_workspace_bytes(head_dim: int, q_tokens: int, q_heads: int) -> int:
    n = int(lib().b200_kv_cache_scores_workspace_bytes(head_dim, q_tokens, q_heads))
    if n < 0:
        raise ValueError(f"no attention kernel for head_dim {head_dim}, {q_heads} heads")
    return n


def kv_cache_scores(q: torch.Tensor, cache, page_table: torch.Tensor, kv_lens: torch.Tensor,
                    q_starts: torch.Tensor, max_q_len: int, lse: torch.Tensor,
                    scores: torch.Tensor, *, scale: float | None = None, causal: bool = True,
                    window: int = 0, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Adds to each cached token's score the attention weight it has from the sequences'
    new tokens, summed over them and the query heads of each key/value head; the new
    tokens' own scores start from zero (``causal=False``: the queries' tokens are not
    among the cached ones, and all scores are added to).

    Call it after the attention call, with its arguments and its log-sum-exp ``lse``.
    ``scores`` fp32 ``[pages, page_size, kv_heads]``, any strides
    (:meth:`~.kv_cache.PagedKVCache.empty_scores`); ``out``, by default ``scores``
    itself, takes the new values. No page may stand twice among those of the call's
    tokens. The result does not depend on timing. Returns ``out``."""
    index = _on_device("kv_cache_scores", q, cache.k, page_table, kv_lens, q_starts, lse, scores,
                       out, workspace)
    code, tokens, heads, dim, seqs, _ = _attention_args(q, cache, page_table, kv_lens, q_starts, q)
    if lse.dtype != torch.float32 or lse.shape != (tokens, heads) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 [{tokens}, {heads}], got {lse.dtype} "
                         f"{tuple(lse.shape)}")
    _scores_of(scores, cache)
    if out is None:
        out = scores
    else:
        _scores_of(out, cache, "out")
    if 0 in q.stride()[:2]:  # one vector for several rows: not for tensor copies
        q = q.contiguous()
    stream = _raw_stream(index)
    if workspace is not None:
        ws = _own_workspace(workspace)
    else:
        key = (dim, -(-tokens // 256) * 256, heads)
        nbytes = _SCORES_BYTES.get(key)
        if nbytes is None:
            nbytes = _SCORES_BYTES[key] = kv_cache_scores_workspace_bytes(*key)
        ws = _attn_workspace_of(index, stream, nbytes)
    _lib.check(lib().b200_kv_cache_scores(
        cache.desc, q.data_ptr(), code, tokens, heads, q.stride(0), q.stride(1),
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1], kv_lens.data_ptr(),
        q_starts.data_ptr(), seqs, max_q_len, dim ** -0.5 if scale is None else scale, causal,
        window, lse.data_ptr(), scores.data_ptr(), *scores.stride(), out.data_ptr(), *out.stride(),
        ws.data_ptr(), ws.numel(), stream))
    return out


def kv_cache_evict(cache, scores: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                   budget: int, *, recent: int = 0, first: int = 0,
                   out_table: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keeps ``budget`` tokens of each sequence and key/value head: the first ``first``,
    the last ``recent``, and of those between the ones with the largest ``scores``
    (fp32 ``[pages, page_size, kv_heads]``, see :func:`kv_cache_scores`; ties: the
    lowest index). Heads choose by themselves; the kept tokens stay in order.

    Without ``out_table`` they move to the front of the sequence's own pages, keys,
    values, scales and scores, in place; no page may stand twice among those tokens' pages.
    With it (int32 ``[seqs, pages]``, pages that hold none of the sequences' tokens)
    they are copied there, and the source stays.

    Returns (kept int32 ``[seqs, kv_heads, budget]``: the tokens' indices before, -1
    past the end; lens int32 ``[seqs]``: ``min(kv_lens, budget)``)."""
    index = _on_device("kv_cache_evict", cache.k, scores, page_table, kv_lens, out_table)
    _scores_of(scores, cache)
    _tables((page_table, "page_table"), (kv_lens, "kv_lens"))
    seqs = kv_lens.shape[0]
    if kv_lens.dim() != 1 or page_table.dim() != 2 or page_table.shape[0] != seqs:
        raise ValueError(f"kv_lens must be [seqs] and page_table [seqs, pages], got "
                         f"{tuple(kv_lens.shape)}, {tuple(page_table.shape)}")
    to = (None, 0, 0)
    if out_table is not None:
        _tables((out_table, "out_table"))
        if out_table.dim() != 2 or out_table.shape[0] != seqs:
            raise ValueError(f"out_table must be [{seqs}, pages], got {tuple(out_table.shape)}")
        to = (out_table.data_ptr(), out_table.stride(0), out_table.shape[1])
    if not 0 < budget < 1 << 31 or recent < 0 or first < 0 or recent + first > budget:
        raise ValueError(f"the budget must be a positive int32 and hold the first and recent tokens, "
                         f"got {budget}, {first}, {recent}")
    kept = torch.empty(seqs, cache.kv_heads, budget, dtype=torch.int32, device=scores.device)
    lens = torch.empty(seqs, dtype=torch.int32, device=scores.device)
    _lib.check(lib().b200_kv_cache_evict(
        cache.desc, scores.data_ptr(), *scores.stride(), page_table.data_ptr(),
        page_table.stride(0), page_table.shape[1], kv_lens.data_ptr(), seqs, budget, recent, first,
        *to, kept.data_ptr(), lens.data_ptr(), _raw_stream(index)))
    return kept, lens
