"""Torch-facing wrappers of the sm_100a kernels (C ABI in include/lbx.h).

These mirror the reference's native op library
(patches/littlebit_cpu_optimized.cpp, ``torch.ops.littlebit_cpu_ops.*``,
schemas at :2321-2377) on CUDA tensors: same argument meaning, same shape
checks, RuntimeError on bad input.  There is no CPU path — CPU tensors are
rejected, and a missing kernel library raises at import of ``_lib``.
"""
from __future__ import annotations

import ctypes
import threading
from dataclasses import dataclass, field
from typing import Optional, Sequence

import torch

from . import _lib as L


# ---------------------------------------------------------------------------
# plumbing
# ---------------------------------------------------------------------------
def lib():
    return L.load()


def _stream(device: torch.device | None = None) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _cuda(name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (the B200 library has no CPU path)")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return L.LBX_F32
    if t.dtype == torch.bfloat16:
        return L.LBX_BF16
    raise RuntimeError(f"unsupported activation dtype {t.dtype} (float32 or bfloat16)")


class Workspace:
    """A growable device scratch buffer (one per device and purpose).

    Zero-filled when (re)allocated: the kernels keep small bookkeeping words in
    the workspace that must start at zero and are left at zero by every call."""

    def __init__(self, device: torch.device):
        self.device = device
        self.buf = torch.zeros(0, dtype=torch.uint8, device=device)

    def get(self, nbytes: int) -> torch.Tensor:
        if self.buf.numel() < nbytes:
            self.buf = torch.zeros(max(nbytes, 2 * self.buf.numel()), dtype=torch.uint8,
                                   device=self.device)
        return self.buf


_WS: dict = {}


def workspace(device: torch.device, tag: str = "op") -> Workspace:
    key = (torch.device(device).index or 0, tag)
    if key not in _WS:
        _WS[key] = Workspace(torch.device(device))
    return _WS[key]


def device_error(device=None) -> int:
    v = ctypes.c_int32(0)
    L.check(lib().lbx_device_error(ctypes.byref(v), _stream(device)), "lbx_device_error")
    return v.value


def clear_device_error(device=None) -> None:
    L.check(lib().lbx_clear_device_error(_stream(device)), "lbx_clear_device_error")


# ---------------------------------------------------------------------------
# bit packing (quantization/utils/binary_packer.py)
# ---------------------------------------------------------------------------
def binary_packer(tensor: torch.Tensor) -> torch.Tensor:
    """±1 int8 [rows, cols] -> int32 [rows, ceil(cols/32)], LSB-first, bit 1 <=> -1
    (binary_packer.py:4-50).  Raises TypeError for non-int8 input like the reference."""
    if tensor.dtype != torch.int8:
        raise TypeError("Input tensor must be int8.")
    _cuda("tensor", tensor)
    if tensor.dim() != 2:
        raise ValueError("binary_packer expects a 2-D tensor")
    rows, cols = tensor.shape
    out = torch.empty(rows, (cols + 31) // 32, dtype=torch.int32, device=tensor.device)
    L.check(lib().lbx_pack_signs(_p(tensor), rows, cols, _p(out), None, _stream(tensor.device)),
            "binary_packer")
    return out


def binary_unpacker(packed_tensor: torch.Tensor, original_shape) -> torch.Tensor:
    """int32 words -> ±1 int8 of ``original_shape`` (binary_packer.py:53-97)."""
    _cuda("packed_tensor", packed_tensor)
    if packed_tensor.dim() == 2:
        n_rows, n_cols = (int(v) for v in original_shape)
        if tuple(packed_tensor.shape) == (n_rows, (n_cols + 31) // 32):
            if packed_tensor.dtype != torch.int32:
                raise TypeError("packed tensor must be int32")
            out = torch.empty(n_rows, n_cols, dtype=torch.int8, device=packed_tensor.device)
            L.check(lib().lbx_unpack_signs(_p(packed_tensor), n_rows, n_cols, _p(out),
                                           _stream(packed_tensor.device)), "binary_unpacker")
            return out
    raise ValueError(f"Unsupported packed tensor format. Expected 2D tensor with shape "
                     f"(n_rows, words_per_row), got {packed_tensor.shape} with "
                     f"{packed_tensor.dim()} dimensions.")


def pack_signs_from_float(w: torch.Tensor) -> torch.Tensor:
    """sign(w) (0 -> +1) packed straight from a float/bf16 latent factor
    (littlebit.py:313-317 pack_param: quantize -> int8 -> binary_packer)."""
    _cuda("w", w)
    rows, cols = w.shape
    out = torch.empty(rows, (cols + 31) // 32, dtype=torch.int32, device=w.device)
    L.check(lib().lbx_pack_signs_from_float(_p(w), _dt(w), rows, cols, _p(out), _stream(w.device)),
            "pack_signs_from_float")
    return out


# ---------------------------------------------------------------------------
# LittleBit linear
# ---------------------------------------------------------------------------
@dataclass
class Branch:
    """One LittleBit factorisation on device.  ``v_sign is None`` means the
    branch reuses branch 0's V-stage (shared-factor residual)."""
    v_sign: Optional[torch.Tensor]  # int32 [rank, ceil(in/32)]
    v2: Optional[torch.Tensor]      # fp32 [in]
    mid: torch.Tensor               # fp32 [rank]
    u_sign: torch.Tensor            # int32 [out, ceil(rank/32)]
    u1: torch.Tensor                # fp32 [out]
    rank: int


class PackedLinear:
    """Device-resident LittleBitLinear (main + optional residual branch + bias)
    with its C descriptor built once."""

    def __init__(self, in_features: int, out_features: int, branches: Sequence[Branch],
                 bias: Optional[torch.Tensor] = None):
        if not 1 <= len(branches) <= 2:
            raise ValueError("1 or 2 branches")
        self.in_features = int(in_features)
        self.out_features = int(out_features)
        self.branches = list(branches)
        self.bias = bias
        for i, b in enumerate(self.branches):
            for nm in ("mid", "u_sign", "u1"):
                _cuda(f"branch{i}.{nm}", getattr(b, nm))
            if b.v_sign is not None:
                _cuda(f"branch{i}.v_sign", b.v_sign)
                _cuda(f"branch{i}.v2", b.v2)
                if tuple(b.v_sign.shape) != (b.rank, (self.in_features + 31) // 32):
                    raise RuntimeError(f"v_sign shape {tuple(b.v_sign.shape)} != "
                                       f"({b.rank}, {(self.in_features + 31) // 32})")
            if tuple(b.u_sign.shape) != (self.out_features, (b.rank + 31) // 32):
                raise RuntimeError(f"u_sign shape {tuple(b.u_sign.shape)} != "
                                   f"({self.out_features}, {(b.rank + 31) // 32})")
        self.device = self.branches[0].u_sign.device
        self.proj = self._build()

    def _build(self) -> L.Proj:
        pr = L.Proj()
        pr.in_features = self.in_features
        pr.out_features = self.out_features
        pr.n_branches = len(self.branches)
        for i, b in enumerate(self.branches):
            br = pr.br[i]
            br.v_sign = _p(b.v_sign)
            br.v2 = _p(b.v2)
            br.mid = _p(b.mid)
            br.u_sign = _p(b.u_sign)
            br.u1 = _p(b.u1)
            br.rank = int(b.rank)
        pr.bias = _p(self.bias)
        return pr

    def packed_bytes(self) -> int:
        """Algorithmic packed-sign bytes (no word padding)."""
        tot = 0
        for b in self.branches:
            if b.v_sign is not None:
                tot += (b.rank * self.in_features + 7) // 8
            tot += (self.out_features * b.rank + 7) // 8
        return tot

    def scale_bytes(self) -> int:
        tot = 0
        for b in self.branches:
            if b.v_sign is not None:
                tot += 4 * self.in_features
            tot += 4 * (b.rank + self.out_features)
        return tot + (4 * self.out_features if self.bias is not None else 0)


def projs_array(projs: Sequence[PackedLinear]):
    arr = (L.Proj * len(projs))()
    for i, p in enumerate(projs):
        arr[i] = p.proj
    return arr


def linear_chain(layers: Sequence[PackedLinear], acts: Sequence[torch.Tensor],
                 ws: Optional[torch.Tensor] = None, arr=None, ptrs=None) -> None:
    """acts[i+1] = layers[i](acts[i]) for every layer, as one persistent program
    (lbx_linear_chain).  All activations [k, features] share one dtype."""
    n = len(layers)
    if len(acts) != n + 1:
        raise ValueError("need len(layers) + 1 activation buffers")
    for i, t in enumerate(acts):
        _cuda(f"acts[{i}]", t)
    k = acts[0].shape[0]
    if arr is None:
        arr = projs_array(layers)
    if ptrs is None:
        ptrs = (ctypes.c_void_p * (n + 1))(*[t.data_ptr() for t in acts])
    need = int(lib().lbx_linear_chain_workspace_size(arr, n, k))
    if ws is None:
        ws = workspace(acts[0].device, "chain").get(need)
    L.check(lib().lbx_linear_chain(arr, n, k, _dt(acts[0]), ptrs, _p(ws), ws.numel(),
                                   _stream(acts[0].device)), "linear_chain")


class FusedChain:
    """A chain of single-projection layers run by the fused chain executor
    (lbx_chain_fused): layer i's U-stage and layer i+1's V-stage partials in
    one launch, bit-identical to running the layers one by one.  The sign
    words are copied once into the executor's layout (lbx_chain_prepare)."""

    def __init__(self, layers: Sequence[PackedLinear]):
        self.layers = list(layers)
        self.arr = projs_array(self.layers)
        n = len(self.layers)
        nb = int(lib().lbx_chain_prepare_size(self.arr, n))
        if nb == 0:
            raise RuntimeError(f"layer chain does not fit the fused chain executor: {L.last_error()}")
        dev = self.layers[0].device
        self.blob = torch.empty(nb // 4, dtype=torch.int32, device=dev)
        L.check(lib().lbx_chain_prepare(self.arr, n, _p(self.blob), nb, _stream(dev)), "chain_prepare")
        self._ws = {}

    def workspace(self, k: int) -> torch.Tensor:
        if k not in self._ws:
            nb = int(lib().lbx_chain_fused_workspace_size(self.arr, len(self.layers), k))
            if nb == 0:
                raise RuntimeError(f"fused chain: {k} tokens unsupported: {L.last_error()}")
            self._ws[k] = torch.empty(nb, dtype=torch.uint8, device=self.layers[0].device)
        return self._ws[k]

    def run(self, acts: Sequence[torch.Tensor], ptrs=None, stream=None) -> None:
        """acts[i+1] = layers[i](acts[i]); all activations [k, features] of one dtype."""
        n = len(self.layers)
        if len(acts) != n + 1:
            raise ValueError("need len(layers) + 1 activation buffers")
        for i, t in enumerate(acts):
            _cuda(f"acts[{i}]", t)
        k = acts[0].shape[0]
        ws = self.workspace(k)
        if ptrs is None:
            ptrs = (ctypes.c_void_p * (n + 1))(*[t.data_ptr() for t in acts])
        st = _stream(acts[0].device) if stream is None else ctypes.c_void_p(stream.cuda_stream)
        L.check(lib().lbx_chain_fused(self.arr, n, k, _dt(acts[0]), ptrs, _p(self.blob), self.blob.numel() * 4,
                                      _p(ws), ws.numel(), st), "chain_fused")


def linear_workspace_bytes(projs: Sequence[PackedLinear], n_tokens: int) -> int:
    return int(lib().lbx_linear_workspace_size(projs_array(projs), len(projs), n_tokens))


def linear_args(projs: Sequence[PackedLinear], x: torch.Tensor, outs: Sequence[torch.Tensor], *,
                prologue: int = L.LBX_PRO_NONE, norm_w: Optional[torch.Tensor] = None,
                eps: float = 1e-6, x2: Optional[torch.Tensor] = None,
                epilogue: int = L.LBX_EPI_STORE, use_pdl: bool = True,
                exec_mode: int = L.LBX_EXEC_AUTO) -> L.LinearArgs:
    """The lbx_linear_args of a call (checked shapes), for callers that issue the
    C-ABI call themselves, e.g. many times over fixed buffers."""
    _cuda("x", x)
    k = x.shape[0]
    a = L.LinearArgs()
    a.n_proj = len(projs)
    a.n_tokens = k
    a.x_dtype = _dt(x)
    a.y_dtype = _dt(outs[0])
    a.prologue = prologue
    a.epilogue = epilogue
    a.eps = float(eps)
    a.use_pdl = 1 if use_pdl else 0
    a.exec = exec_mode
    a.x = _p(x)
    a.x2 = _p(x2)
    a.norm_w = _p(norm_w)
    for i, o in enumerate(outs):
        _cuda(f"out{i}", o)
        if o.shape[0] != k or o.shape[-1] != projs[i].out_features:
            raise RuntimeError(f"out{i} has shape {tuple(o.shape)}, expected ({k}, {projs[i].out_features})")
        a.y[i] = _p(o)
        a.y_ld[i] = o.stride(0)
    return a


def linear_group(projs: Sequence[PackedLinear], x: torch.Tensor, outs: Sequence[torch.Tensor], *,
                 prologue: int = L.LBX_PRO_NONE, norm_w: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, x2: Optional[torch.Tensor] = None,
                 epilogue: int = L.LBX_EPI_STORE, use_pdl: bool = True,
                 ws: Optional[torch.Tensor] = None, arr=None,
                 exec_mode: int = L.LBX_EXEC_AUTO) -> None:
    """Run 1..3 LittleBit projections that share the input x [k, in].

    ``exec_mode``: LBX_EXEC_AUTO (one cluster launch when the call fits it,
    else the two stage grids), LBX_EXEC_KERNELS or LBX_EXEC_CLUSTER; all give
    the same bits."""
    a = linear_args(projs, x, outs, prologue=prologue, norm_w=norm_w, eps=eps, x2=x2, epilogue=epilogue,
                    use_pdl=use_pdl, exec_mode=exec_mode)
    k = x.shape[0]
    if arr is None:
        arr = projs_array(projs)
    need = int(lib().lbx_linear_workspace_size(arr, len(projs), k))
    if ws is None:
        ws = workspace(x.device, "linear").get(need)
    L.check(lib().lbx_linear_verify(arr, ctypes.byref(a), _p(ws), ws.numel(), _stream(x.device)),
            "littlebit_linear")


def lb_linear(layer: PackedLinear, x: torch.Tensor, out: Optional[torch.Tensor] = None,
              out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y = LittleBitLinear(x) for x [..., in] (float32 or bfloat16)."""
    shp = x.shape
    x2d = x.reshape(-1, shp[-1]).contiguous()
    if out is None:
        out = torch.empty(x2d.shape[0], layer.out_features, dtype=out_dtype, device=x.device)
    linear_group([layer], x2d, [out])
    return out.reshape(*shp[:-1], layer.out_features)


def littlebit_linear(input: torch.Tensor, v2: torch.Tensor, v_sign: torch.Tensor, v_cols: int,
                     mid: torch.Tensor, u_sign: torch.Tensor, u_cols: int, u1: torch.Tensor) -> torch.Tensor:
    """CUDA counterpart of littlebit_cpu_ops.littlebit_linear (cpp:598-701), same
    argument checks, fp32 [M, N] output; no int8 activation quantisation."""
    for nm, t in (("input", input), ("v2", v2), ("mid", mid), ("u1", u1)):
        _cuda(nm, t)
        if t.dtype != torch.float32:
            raise RuntimeError(f"{nm} must be float32")
    for nm, t in (("v_sign", v_sign), ("u_sign", u_sign)):
        _cuda(nm, t)
        if t.dtype != torch.int32:
            raise RuntimeError(f"{nm} must be int32")
    if input.dim() != 2:
        raise RuntimeError("input must have shape [M, K]")
    if not (v2.dim() == 2 and v2.shape[0] == 1):
        raise RuntimeError("v2 must have shape [1, K]")
    if not (mid.dim() == 2 and mid.shape[0] == 1):
        raise RuntimeError("mid must have shape [1, R]")
    if not (u1.dim() == 2 and u1.shape[0] == 1):
        raise RuntimeError("u1 must have shape [1, N]")
    if input.shape[1] != v_cols or v2.shape[1] != v_cols:
        raise RuntimeError("input K must match v_cols")
    if v_sign.dim() != 2 or u_sign.dim() != 2:
        raise RuntimeError("v_sign / u_sign must be 2-D")
    if v_sign.shape[0] != mid.shape[1] or mid.shape[1] != u_cols:
        raise RuntimeError("mid rank must match v_sign rows and u_cols")
    if u_sign.shape[0] != u1.shape[1]:
        raise RuntimeError("u1 out_features must match u_sign rows")
    if v_sign.shape[1] != (v_cols + 31) // 32 or u_sign.shape[1] != (u_cols + 31) // 32:
        raise RuntimeError("packed word counts must equal ceil(cols / 32)")
    layer = PackedLinear(v_cols, u_sign.shape[0],
                         [Branch(v_sign, v2.reshape(-1), mid.reshape(-1), u_sign, u1.reshape(-1), u_cols)])
    out = torch.empty(input.shape[0], layer.out_features, dtype=torch.float32, device=input.device)
    linear_group([layer], input, [out])
    return out


# ---------------------------------------------------------------------------
# decoder pieces (CUDA counterparts of the CPU ops at cpp:973-1301)
# ---------------------------------------------------------------------------
def embedding_lookup(weight: torch.Tensor, indices: torch.Tensor) -> torch.Tensor:
    """weight [vocab, hidden] bf16 (or fp32, converted once), indices [N] or [1, N]
    -> fp32 [N, hidden]  (cpp:973-996)."""
    _cuda("weight", weight)
    if weight.dtype != torch.bfloat16:
        weight = weight.to(torch.bfloat16)
    idx = indices.reshape(-1).to(device=weight.device, dtype=torch.int64).contiguous()
    out = torch.empty(idx.numel(), weight.shape[1], dtype=torch.float32, device=weight.device)
    L.check(lib().lbx_embed(_p(weight), _p(idx), idx.numel(), weight.shape[1], weight.shape[0],
                            _p(out), _stream(weight.device)), "embedding_lookup")
    return out


def rms_norm(input: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """x * rsqrt(mean(x^2) + eps) * w over the last dim; any number of rows
    (the CPU op accepts one row, cpp:998-1052)."""
    _cuda("input", input)
    _cuda("weight", weight)
    h = weight.numel()
    x = input.reshape(-1, h)
    out = torch.empty_like(x, dtype=torch.float32)
    L.check(lib().lbx_rmsnorm(_p(x), _p(weight), x.shape[0], h, float(eps), _p(out),
                              _stream(input.device)), "rms_norm")
    return out


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """SiLU(gate) * up (cpp:1117-1170), exact exp."""
    _cuda("gate", gate)
    _cuda("up", up)
    if gate.shape != up.shape:
        raise RuntimeError("gate and up must have same shape")
    out = torch.empty_like(gate)
    L.check(lib().lbx_silu_mul(_p(gate), _p(up), gate.numel(), _p(out), _stream(gate.device)),
            "silu_mul")
    return out


def rope_(x: torch.Tensor, pos: torch.Tensor, heads: int, head_dim: int, theta: float) -> torch.Tensor:
    """In-place HF-Llama rotary embedding on x [n, heads*head_dim] at positions pos [n]."""
    _cuda("x", x)
    p = pos.to(device=x.device, dtype=torch.int32).contiguous()
    L.check(lib().lbx_rope(_p(x), _p(p), x.shape[0], heads, head_dim, float(theta),
                           _stream(x.device)), "rope")
    return x


def dense_gemv_f32(input: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """lm_head GEMV (cpp:1054-1115): input [n, K] fp32, weight [N, K] bf16 -> fp32 [n, N]."""
    _cuda("input", input)
    _cuda("weight", weight)
    if weight.dtype != torch.bfloat16:
        raise RuntimeError("weight must be bfloat16 on the B200 path")
    if input.shape[-1] != weight.shape[1]:
        raise RuntimeError("input K must match weight K")
    x = input.reshape(-1, weight.shape[1]).to(torch.float32).contiguous()
    out = torch.empty(x.shape[0], weight.shape[0], dtype=torch.float32, device=x.device)
    ws = workspace(x.device, "lm").get(int(lib().lbx_lmhead_workspace_size(x.shape[0], weight.shape[0])))
    L.check(lib().lbx_lmhead_argmax(_p(x), None, 0.0, x.shape[0], weight.shape[1], _p(weight),
                                    weight.shape[0], _p(out), None, _p(ws), ws.numel(), 0,
                                    _stream(x.device)), "dense_gemv_f32")
    return out


def lmhead_argmax(x: torch.Tensor, weight: torch.Tensor, norm_w: Optional[torch.Tensor] = None,
                  eps: float = 1e-6, want_logits: bool = True):
    """Fused final RMSNorm + lm_head + argmax.  Returns (logits or None, argmax int64 [n])."""
    _cuda("x", x)
    _cuda("weight", weight)
    n = x.shape[0]
    logits = (torch.empty(n, weight.shape[0], dtype=torch.float32, device=x.device)
              if want_logits else None)
    am = torch.empty(n, dtype=torch.int64, device=x.device)
    ws = workspace(x.device, "lm").get(int(lib().lbx_lmhead_workspace_size(n, weight.shape[0])))
    L.check(lib().lbx_lmhead_argmax(_p(x), _p(norm_w), float(eps), n, weight.shape[1], _p(weight),
                                    weight.shape[0], _p(logits), _p(am), _p(ws), ws.numel(), 0,
                                    _stream(x.device)), "lmhead_argmax")
    return logits, am


def attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, pos: torch.Tensor,
              k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_len: int, heads: int,
              kv_heads: int, head_dim: int, scale: float, theta: float,
              tree_mask: Optional[torch.Tensor] = None,
              rope_cs: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention for n new tokens (RoPE + bf16 KV write + causal/tree mask).
    ``rope_cs``: the (cos, sin) table of ``pos`` from :func:`rope_table` (the
    kernel evaluates the same values itself when it is None)."""
    for nm, t in (("q", q), ("k_new", k_new), ("v_new", v_new), ("k_cache", k_cache),
                  ("v_cache", v_cache)):
        _cuda(nm, t)
    n = q.shape[0]
    a = L.AttnArgs()
    a.n = n
    a.heads, a.kv_heads, a.head_dim = heads, kv_heads, head_dim
    a.max_seq = k_cache.shape[1]
    a.prefix_len = int(prefix_len)
    a.scale, a.theta = float(scale), float(theta)
    a.use_pdl = 0
    p32 = pos.to(device=q.device, dtype=torch.int32).contiguous()
    a.q, a.q_ld = _p(q), q.stride(0)
    a.k_new, a.v_new, a.kv_ld = _p(k_new), _p(v_new), k_new.stride(0)
    a.pos = _p(p32)
    tm = None
    if tree_mask is not None:
        tm = tree_mask.to(device=q.device, dtype=torch.int64).contiguous()
    a.tree_mask = _p(tm)
    a.k_cache, a.v_cache = _p(k_cache), _p(v_cache)
    if rope_cs is not None:
        _cuda("rope_cs", rope_cs)
        if rope_cs.dtype != torch.float32 or rope_cs.numel() != n * head_dim or not rope_cs.is_contiguous():
            raise RuntimeError("rope_cs must be a contiguous float32 [n, head_dim] table from rope_table")
        a.rope_cs = _p(rope_cs)
    out = torch.empty(n, heads * head_dim, dtype=torch.float32, device=q.device)
    a.out = _p(out)
    ws = workspace(q.device, "attn").get(int(lib().lbx_attn_workspace_size(ctypes.byref(a))))
    L.check(lib().lbx_attn_decode(ctypes.byref(a), _p(ws), ws.numel(), _stream(q.device)),
            "attention")
    return out


def rope_table(pos: torch.Tensor, head_dim: int, theta: float) -> torch.Tensor:
    """(cos, sin) of pos[i] * theta^(-2j/head_dim) for j < head_dim/2 as a float32
    [n, head_dim] table (pairs), for :func:`attention`'s ``rope_cs``."""
    _cuda("pos", pos)
    p32 = pos.to(dtype=torch.int32).contiguous()
    n = p32.numel()
    out = torch.empty(n, head_dim, dtype=torch.float32, device=pos.device)
    L.check(lib().lbx_rope_table(_p(p32), n, head_dim, float(theta), _p(out), _stream(pos.device)),
            "rope_table")
    return out


def accept_greedy_chain(draft: torch.Tensor, target_argmax: torch.Tensor) -> torch.Tensor:
    """-> int64 [2] = (accepted count, next token) on device."""
    out = torch.empty(2, dtype=torch.int64, device=target_argmax.device)
    L.check(lib().lbx_accept_greedy_chain(_p(draft), _p(target_argmax), draft.numel(), _p(out),
                                          _stream(out.device)), "accept_greedy_chain")
    return out


def accept_greedy_tree(cand: torch.Tensor, node_argmax: torch.Tensor,
                       retrieve: torch.Tensor) -> torch.Tensor:
    """-> int64 [3 + D] = (best row, accept length, bonus token, accepted node ids...)."""
    L_, D1 = retrieve.shape
    out = torch.empty(3 + D1 - 1, dtype=torch.int64, device=cand.device)
    L.check(lib().lbx_accept_greedy_tree(_p(cand), _p(node_argmax), _p(retrieve), L_, D1, _p(out),
                                         _stream(out.device)), "accept_greedy_tree")
    return out


# ---------------------------------------------------------------------------
# 8-bit integer product (scales for each token and each channel)
# ---------------------------------------------------------------------------
_FLOATS = (torch.float32, torch.bfloat16)
_DTYPE = {torch.float32: L.LBX_F32, torch.bfloat16: L.LBX_BF16}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda i: torch.cuda.current_stream(i).cuda_stream)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


def _rows(name: str, t: torch.Tensor, dtypes=_FLOATS) -> torch.Tensor:
    """A 2-D CUDA tensor whose rows are contiguous (any row stride that does not overlap)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (the B200 library has no CPU path)")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name} has type {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if t.is_contiguous() and t.dim() == 2:
        return t
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise RuntimeError(f"{name} must be 2-D with contiguous rows, got shape {tuple(t.shape)} strides {t.stride()}")
    return t


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _vec(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, index: int) -> int:
    """Address of a contiguous tensor of n values on device ``index``."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype or t.numel() != n or t.get_device() != index or not t.is_contiguous():
        raise RuntimeError(f"{name} must hold {n} contiguous {dtype} values on cuda:{index}, got {tuple(t.shape)} "
                           f"{t.dtype} on {t.device}")
    return t.data_ptr()


class _on:
    """Makes a device current for a call where it is not; gives its current stream."""
    __slots__ = ("index", "prev")

    def __init__(self, index: int):
        self.index, self.prev = index, None

    def __enter__(self) -> int:
        cur = torch._C._cuda_getDevice()
        if cur != self.index:
            self.prev = cur
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)


class _Scratch(Workspace):
    """Scratch of one operator on one stream (calls on different streams never share it).
    Its lock is held from :meth:`take` until the call's launches are in the stream: a call
    is several launches that pass results through the scratch, and another thread's on the
    same stream must not come between them (the C call lets other threads run)."""

    def __init__(self, device: torch.device):
        super().__init__(device)
        self.lock = threading.RLock()  # (a finaliser that calls the operator finds its own thread's)

    def take(self, nbytes: int, zeros: int = 0) -> torch.Tensor:
        """The scratch, for the holder of the lock.  A captured call has its own, of the
        graph's memory (it lives as long as the graph, whatever later calls need), its
        first ``zeros`` bytes set by the graph."""
        if _capturing():
            buf = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            buf[:zeros].zero_()
            return buf
        buf = self.buf
        return buf if buf.numel() >= nbytes else self.get(nbytes)


_SCRATCH: dict = {}


def _stream_ws(index: int, tag: str, stream: int) -> _Scratch:
    key = (index, tag, stream)
    # (of two threads that come first, both get the one that is kept)
    return _SCRATCH.get(key) or _SCRATCH.setdefault(key, _Scratch(torch.device("cuda", index)))


def quantize_tokens(x: torch.Tensor):
    """x [m, k] (float32 or bfloat16) -> (codes int8 [m, k], scale float32 [m]): each
    row in 8 bits by its absolute maximum.  Rows of the codes start on 16 bytes,
    as :func:`linear_int8` wants its weights: ``quantize_tokens(weight)`` quantises a
    weight matrix by output channel."""
    _rows("x", x)
    m, k = x.shape
    ld = -(-k // 16) * 16
    q = torch.empty(m, ld, dtype=torch.int8, device=x.device)[:, :k]
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    with _on(x.get_device()) as st:
        L.check(lib().lbx_quant_tokens(x.data_ptr(), _DTYPE[x.dtype], _ld(x), m, k, q.data_ptr(), ld,
                                       scale.data_ptr(), st), "quantize_tokens")
    return q, scale


def linear_int8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y[t, n] = s_t * weight_scale[n] * sum_k c_tk * weight[n, k] (+ bias[n]).

    x [m, k] float32 or bfloat16 is quantised by token in the call (c, s of
    :func:`quantize_tokens`); weight int8 [n, k] has rows on 16 bytes.  The sums
    are exact integers, so a token's result does not depend on the others.
    Result type: ``out_dtype``, else x's."""
    _rows("x", x)
    _rows("weight", weight, (torch.int8,))
    (m, k), (n, kw) = x.shape, weight.shape
    if kw != k:
        raise RuntimeError(f"x has {k} features, weight {kw}")
    dev = x.get_device()
    if weight.get_device() != dev:
        raise RuntimeError("x and weight must be on one device")
    if out is None:
        out = torch.empty(m, n, dtype=out_dtype or x.dtype, device=x.device)
    else:
        _rows("out", out)
        if tuple(out.shape) != (m, n) or out.get_device() != dev or (out_dtype is not None and out.dtype != out_dtype):
            raise RuntimeError(f"out must be [{m}, {n}] on cuda:{dev}")
    if out.dtype not in _FLOATS:
        raise RuntimeError(f"unsupported result type {out.dtype} (float32 or bfloat16)")
    a = L.Int8Args(m, n, k, _DTYPE[x.dtype], _DTYPE[out.dtype], 1, x.data_ptr(), _ld(x), weight.data_ptr(),
                   _ld(weight), _vec("weight_scale", weight_scale, n, torch.float32, dev),
                   None if bias is None else _vec("bias", bias, n, torch.float32, dev), out.data_ptr(), _ld(out))
    with _on(dev) as st:
        c, sc = lib(), _stream_ws(dev, "int8", st)
        with sc.lock:
            ws = sc.take(c.lbx_linear_int8_workspace_size(m, n, k), L.LBX_INT8_TICKET_BYTES)
            L.check(c.lbx_linear_int8(ctypes.byref(a), ws.data_ptr(), ws.numel(), st), "linear_int8")
    return out


class Int8Linear:
    """A dense layer (an lm_head, say) kept as 8-bit integers with a scale for each
    output channel: half the bytes of bf16 for every token that reads it."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None):
        self.weight, self.weight_scale, self.bias = weight, weight_scale, bias

    @classmethod
    def from_float(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> "Int8Linear":
        """Quantise weight [out, in] (float32 or bfloat16) by output channel."""
        q, s = quantize_tokens(weight)
        return cls(q, s, None if bias is None else bias.to(torch.float32).contiguous())

    @property
    def out_features(self) -> int:
        return self.weight.shape[0]

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return linear_int8(x, self.weight, self.weight_scale, self.bias, out, out_dtype)


# ---------------------------------------------------------------------------
# KV cache held in 4 bits
# ---------------------------------------------------------------------------
KV4_GROUP = 64


class Kv4Cache:
    """Keys and values of S sequences in 4 bits: codes uint8 [S, kv_heads, max_seq,
    head_dim / 2] and, for each group of 64 dimensions, (step, least) bfloat16
    [S, kv_heads, max_seq, head_dim / 64, 2]; a value is least + step * code.
    The order of the codes is that of include/lbx.h; :func:`kv4_read` gives the
    values back.  A cache's tensors are fixed: its C descriptor is made once."""
    __slots__ = ("k_codes", "k_params", "v_codes", "v_params", "index", "_struct")

    def __init__(self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor):
        kc, kp, vc, vp = k_codes, k_params, v_codes, v_params
        for t, ty in ((kc, torch.uint8), (vc, torch.uint8), (kp, torch.bfloat16), (vp, torch.bfloat16)):
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is ty and t.is_contiguous()):
                raise RuntimeError("codes must be contiguous uint8 CUDA tensors and params bfloat16 ones (the B200 "
                                   "library has no CPU path)")
        index = kc.get_device()
        if not index == kp.get_device() == vc.get_device() == vp.get_device():
            raise RuntimeError("cache tensors must be on one device")
        shape, pshape = kc.shape, kp.shape
        if len(shape) != 4 or len(pshape) != 5:
            raise RuntimeError("codes must be 4-D and params 5-D")
        S, H, T, D2 = shape
        if vc.shape != shape or vp.shape != pshape or pshape != (S, H, T, 2 * D2 // KV4_GROUP, 2):
            raise RuntimeError(f"cache shapes do not fit together: {tuple(kc.shape)} {tuple(kp.shape)} "
                               f"{tuple(vc.shape)} {tuple(vp.shape)}")
        self.k_codes, self.k_params, self.v_codes, self.v_params, self.index = kc, kp, vc, vp, index
        self._struct = L.Kv4Cache(kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(), S, H, T, 2 * D2)

    @classmethod
    def empty(cls, n_seq: int, kv_heads: int, max_seq: int, head_dim: int, device="cuda") -> "Kv4Cache":
        """max_seq is rounded up to a multiple of 64."""
        if head_dim not in (64, 128):
            raise RuntimeError("head_dim must be 64 or 128")
        shp = (n_seq, kv_heads, -(-max_seq // 64) * 64)
        c = [torch.zeros(*shp, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2)]
        p = [torch.zeros(*shp, head_dim // KV4_GROUP, 2, dtype=torch.bfloat16, device=device) for _ in range(2)]
        return cls(c[0], p[0], c[1], p[1])

    @property
    def shape(self):
        """(n_seq, kv_heads, max_seq, head_dim)"""
        s = self.k_codes.shape
        return s[0], s[1], s[2], 2 * s[3]

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_params, self.v_codes, self.v_params))

    def struct(self) -> L.Kv4Cache:
        """The C descriptor."""
        return self._struct


def _start_arg(name: str, start, n_seq: int, bound: Optional[int], last: int, index: int):
    """(device address or None, host bound) of per-sequence slot counts: an int for all,
    or a device int32 [n_seq] with its host-side upper bound (``last``, the last slot that
    the call's tokens fit at, where the caller names none)."""
    if isinstance(start, torch.Tensor):
        return _vec(name, start, n_seq, torch.int32, index), last if bound is None else int(bound)
    return None, int(start)


def kv4_append(k_new: torch.Tensor, v_new: torch.Tensor, cache: Kv4Cache, start, max_start: Optional[int] = None,
               rope_cs: Optional[torch.Tensor] = None) -> None:
    """Rotate (keys, by ``rope_cs`` of :func:`rope_table`), quantise and store n new
    tokens of every sequence of the cache.

    k_new / v_new [S * n, kv_heads * head_dim], float32 or bfloat16, sequence by
    sequence.  ``start``: first slot, an int for every sequence, or a device int32
    [S] bounded by ``max_start`` (None: the last slot that the tokens fit at)."""
    c, dev = cache.struct(), cache.index
    _rows("k_new", k_new)
    _rows("v_new", v_new, (k_new.dtype,))
    rows, width = k_new.shape
    if v_new.shape != k_new.shape or width != c.kv_heads * c.head_dim or rows % c.n_seq:
        raise RuntimeError(f"k_new / v_new must be [{c.n_seq} * n, {c.kv_heads * c.head_dim}], got "
                           f"{tuple(k_new.shape)} and {tuple(v_new.shape)}")
    if k_new.get_device() != dev or v_new.get_device() != dev:
        raise RuntimeError("k_new, v_new and the cache must be on one device")
    ld = _ld(k_new)
    if rows > 1 and _ld(v_new) != ld:
        raise RuntimeError("k_new and v_new must have one row stride")
    sp, bound = _start_arg("start", start, c.n_seq, max_start, c.max_seq - rows // c.n_seq, dev)
    rope = None if rope_cs is None else _vec("rope_cs", rope_cs, rows * c.head_dim, torch.float32, dev)
    a = L.Kv4AppendArgs(c, rows // c.n_seq, bound, _DTYPE[k_new.dtype], 1, sp, k_new.data_ptr(), v_new.data_ptr(), ld,
                        rope)
    with _on(dev) as st:
        L.check(lib().lbx_kv4_append(ctypes.byref(a), st), "kv4_append")


def kv4_read(cache: Kv4Cache, start, max_start: Optional[int], n: int):
    """The values of n slots of every sequence: (k, v) float32 [S, kv_heads, n, head_dim].
    ``start`` and ``max_start`` as of :func:`kv4_append`."""
    c, dev = cache.struct(), cache.index
    sp, bound = _start_arg("start", start, c.n_seq, max_start, c.max_seq - n, dev)
    kv = torch.empty(2, c.n_seq, c.kv_heads, n, c.head_dim, dtype=torch.float32, device=cache.k_codes.device)
    k, v = kv.unbind(0)
    with _on(dev) as st:
        L.check(lib().lbx_kv4_read(ctypes.byref(c), sp, bound, n, k.data_ptr(), v.data_ptr(), st), "kv4_read")
    return k, v


def attention_kv4(q: torch.Tensor, cache: Kv4Cache, prefix, max_prefix: Optional[int], heads: int, scale: float,
                  rope_cs: Optional[torch.Tensor] = None, tree_mask: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of n new tokens of every sequence over its 4-bit cache, which
    already holds them (:func:`kv4_append`).

    q [S * n, heads * head_dim], float32 or bfloat16, is rotated by ``rope_cs``.
    ``prefix``: cached slots before the new tokens, an int, or a device int32 [S]
    bounded by ``max_prefix`` (None: as many as leave room for the new tokens; a near bound
    makes a smaller grid).  A query sees its sequence's cached slots and the
    new ones up to itself, or those of its ``tree_mask`` bits (int64 [S * n], n <= 64).
    A query that sees nothing gives zeros.  Result: q's shape and type.

    float32 calls hold queries and weights in 22 bits, bfloat16 calls in 11 (their result
    has 8); sums are float32 in both."""
    c, dev = cache.struct(), cache.index
    _rows("q", q)
    rows, width = q.shape
    if q.get_device() != dev:
        raise RuntimeError("q and the cache must be on one device")
    if rows == 0 or rows % c.n_seq or width != heads * c.head_dim:
        raise RuntimeError(f"q must be [{c.n_seq} * n, {heads * c.head_dim}], got {tuple(q.shape)}")
    pp, bound = _start_arg("prefix", prefix, c.n_seq, max_prefix, c.max_seq - rows // c.n_seq, dev)
    rope = None if rope_cs is None else _vec("rope_cs", rope_cs, rows * c.head_dim, torch.float32, dev)
    tm = None if tree_mask is None else _vec("tree_mask", tree_mask, rows, torch.int64, dev)
    if out is None:
        out = torch.empty((rows, width), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous():
        raise RuntimeError("out must be contiguous, with q's shape, type and device")
    a = L.Kv4AttnArgs(c, rows // c.n_seq, heads, bound, _DTYPE[q.dtype], 1, scale, pp, q.data_ptr(), _ld(q), rope, tm,
                      out.data_ptr())
    with _on(dev) as st:
        cl, sc = lib(), _stream_ws(dev, "kv4", st)
        ref = ctypes.byref(a)
        with sc.lock:
            ws = sc.take(cl.lbx_kv4_attn_workspace_size(ref) or 1)
            L.check(cl.lbx_kv4_attn(ref, ws.data_ptr(), ws.numel(), st), "attention_kv4")
    return out


# ---------------------------------------------------------------------------
# verification of sampled drafts
# ---------------------------------------------------------------------------
def accept_sampled(tokens: Optional[torch.Tensor], target_logits: torch.Tensor, draft_logits: Optional[torch.Tensor],
                   u: Optional[torch.Tensor], e: torch.Tensor, temperature=1.0,
                   n_draft: Optional[torch.Tensor] = None):
    """Verify k sampled drafts of each of S sequences (speculative_decoding.py:331-363)
    from given random numbers -> (accepted int64 [S], next token int64 [S]).

    tokens int64 [S, k]; target_logits [S, k + 1, V] and draft_logits [S, k, V],
    float32 or bfloat16 (draft_logits None: the drafts were not sampled); u float32
    [S, k] uniform in [0, 1); e float32 [S, V] exponentially distributed (> 0);
    temperature a number or a device float32 [S]; n_draft int32 [S]: sequences
    with fewer drafts.  With k = 0 (tokens, draft_logits and u None or empty) it
    draws next from softmax(target_logits[:, 0] / temperature)."""
    t = target_logits
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 3 or t.dtype not in _FLOATS:
        raise RuntimeError("target_logits must be a float32 or bfloat16 CUDA tensor [S, k + 1, V]")
    S, k1, V = t.shape
    k, dev = k1 - 1, t.get_device()
    if k < 0 or V < 1:
        raise RuntimeError("target_logits must be [S, k + 1, V] with V >= 1")

    def plane(name, x, shape, dtype):
        if not isinstance(x, torch.Tensor) or x.get_device() != dev:
            raise RuntimeError(f"{name} must be a tensor on cuda:{dev}")
        if x.shape != shape or x.dtype is not dtype:
            raise RuntimeError(f"{name} must be {shape} {dtype}, got {tuple(x.shape)} {x.dtype}")
        st = x.stride()
        if st[-1] != 1 and shape[-1] > 1:
            raise RuntimeError(f"{name} must be contiguous along its last dimension")
        return x.data_ptr(), *st[:-1]

    tp = plane("target_logits", t, (S, k1, V), t.dtype)
    ep = plane("e", e, (S, V), torch.float32)
    tk, up, dp, nd, temps = (None, 0), (None, 0), (None, 0, 0), None, None
    if k:
        tk = plane("tokens", tokens, (S, k), torch.int64)
        up = plane("u", u, (S, k), torch.float32)
        if draft_logits is not None:
            dp = plane("draft_logits", draft_logits, (S, k, V), t.dtype)
        if n_draft is not None:
            nd = _vec("n_draft", n_draft, S, torch.int32, dev)
    if isinstance(temperature, torch.Tensor):
        temps, temperature = _vec("temperature", temperature, S, torch.float32, dev), 0.0
    res = torch.empty((2, S), dtype=torch.int64, device=t.device)
    rp = res.data_ptr()
    a = L.AcceptArgs(S, k, V, _DTYPE[t.dtype], 1, temperature, temps, *tk, nd, *tp, *dp, *up, *ep, rp, rp + 8 * S)
    with _on(dev) as st:
        L.check(lib().lbx_accept_sampled(ctypes.byref(a), st), "accept_sampled")
    return res.unbind(0)
