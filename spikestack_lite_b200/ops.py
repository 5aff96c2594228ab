"""Tensor-level ops over the C ABI (torch tensors in, torch tensors out).

Every op validates its tensors (CUDA, float32, contiguous where the kernel
needs it), passes raw pointers and the current stream of the tensors' device
to libspk_b200.so and raises ``EngineError`` (a RuntimeError) on any failure.
"""
import functools
import weakref

import torch

from . import _lib
from ._lib import EngineError, check, ptr, require_cuda, require_f32, stream_of


def _branch(b):
    if isinstance(b, int):
        return b
    try:
        return _lib.BRANCHES[b]
    except KeyError:
        raise EngineError(f"unknown branch {b!r} (auto, dense or csr)") from None


def _contig(t):
    return t if t.is_contiguous() else t.contiguous()


# (op, rows, K, N) of every dense contraction issued while a tally is open
_TALLY = None


class tally:
    """Records (op, rows, K, N) of each tensor-core contraction the ops issue
    inside the ``with`` block -- spike_linear, linear_act and the recurrent
    projections of gsmc_forward -- so that a caller can count their
    algorithmic FLOPs (2 * rows * K * N each).  Bookkeeping only."""

    def __enter__(self):
        global _TALLY
        self.calls = []
        _TALLY = self.calls
        return self

    def __exit__(self, *exc):
        global _TALLY
        _TALLY = None
        return False

    def flops(self):
        return sum(2.0 * r * k * n for _, r, k, n in self.calls)


def _record(op, rows, K, N):
    if _TALLY is not None:
        _TALLY.append((op, int(rows), int(K), int(N)))


# ------------------------------------------------------------ prepared weights
# The dense branch reads W through a weight image (spk_weight_image) that the
# plain entry points rebuild from W on every call.  Weights that stay fixed
# between calls (inference) get theirs built once: the cache holds one image
# per live weight tensor, valid while the tensor object, its version counter
# (bumped by every in-place change), pointer, shape, strides and dtype are
# unchanged, and drops it when the tensor is freed.  A weight changed through
# `.data` escapes the version counter: call clear_weight_cache() after that.
_IMG = {}
_IMG_ENABLED = True


def set_weight_cache(enabled):
    """Turn the prepared-weight cache on or off (on by default)."""
    global _IMG_ENABLED
    _IMG_ENABLED = bool(enabled)
    if not _IMG_ENABLED:
        _IMG.clear()


def clear_weight_cache():
    _IMG.clear()


def _weight_image(W, K, N, sk, sn, wdt):
    """The cached weight image of W (a 1024-byte aligned uint8 view), or None
    (cache off, or a stream capture in progress: an image built there would
    hold nothing until the graph is replayed)."""
    if not _IMG_ENABLED:
        return None
    key = (W.data_ptr(), tuple(W.shape), tuple(W.stride()), W.dtype, int(sk), int(sn), int(K), int(N))
    ent = _IMG.get(id(W))
    if ent is not None:
        ref, ver, k, img = ent
        if ref() is W and ver == W._version and k == key:
            return img
    if torch.cuda.is_current_stream_capturing():
        return None
    lib = _lib.load()
    nbytes = int(lib.spk_weight_image_bytes(K, N, wdt))
    buf = torch.empty(nbytes + 1024, dtype=torch.uint8, device=W.device)
    off = (-buf.data_ptr()) % 1024
    img = buf[off:off + nbytes]
    check(lib.spk_weight_image(ptr(W), wdt, sk, sn, K, N, ptr(img), nbytes, stream_of(W)), "spk_weight_image")
    wid = id(W)
    _IMG[wid] = (weakref.ref(W, lambda _r, i=wid: _IMG.pop(i, None)), W._version, key, img)
    return img


# ----------------------------------------------------------------- spike -> CSR
def csr_compact(S, values=True, capacity=None):
    """Per-plane CSR of S [T, M, K] (or [M, K] as one plane).

    Returns a dict with nnz_row [T, M], row_ptr [T, M+1] (int32, relative to
    each plane), col_idx (int32, planes back to back), values (float32 or
    None) and plane_ptr [T+1] (int64).  One launch for all planes, into
    buffers of `capacity` entries (default T*M*K, enough for any input), then
    an 8-byte device->host read of the total to size the returned views."""
    require_cuda(S, what="csr_compact")
    require_f32(S, what="csr_compact")
    S = _contig(S)
    if S.dim() == 2:
        S = S.unsqueeze(0)
    T, M, K = S.shape
    lib = _lib.load()
    dev = S.device
    nnz_row = torch.empty(T, M, dtype=torch.int32, device=dev)
    row_ptr = torch.empty(T, M + 1, dtype=torch.int32, device=dev)
    plane_ptr = torch.empty(T + 1, dtype=torch.int64, device=dev)
    cap = int(capacity) if capacity is not None else T * M * K
    col_idx = torch.empty(max(cap, 1), dtype=torch.int32, device=dev)
    vals = torch.empty(max(cap, 1), dtype=torch.float32, device=dev) if values else None
    ws, wsn = _lib.workspace(dev, lib.spk_csr_workspace_bytes(T, M, K))
    check(lib.spk_csr_compact(ptr(S), T, M, K, ptr(nnz_row), ptr(row_ptr), ptr(col_idx), ptr(vals),
                              ptr(plane_ptr), cap, ws, wsn, stream_of(S)), "spk_csr_compact")
    nnz = int(plane_ptr[T].item())
    if nnz > cap:
        raise EngineError(f"csr_compact: {nnz} spikes exceed the capacity of {cap}")
    return {"nnz_row": nnz_row, "row_ptr": row_ptr, "col_idx": col_idx[:nnz],
            "values": None if vals is None else vals[:nnz], "plane_ptr": plane_ptr}


# ------------------------------------------------------------------ spike-linear
def spike_linear(S, weight=None, weightT=None, bias=None, branch="auto", csr=None):
    """Y[..., n] = sum_{k: S[..., k] > 0} S[..., k] W[k, n] (+ bias) for S [T, M, K]
    (or [M, K]).  W is given either as an nn.Linear ``weight`` [N, K] or as
    ``weightT`` [K, N] (the reference op layout), float32 or bfloat16.

    ``csr``: None, or a dict with preallocated int32/int64 buffers
    {nnz_row [T*M], row_ptr [T*(M+1)], col_idx [cap], plane_ptr [T+1],
    values [cap] (optional)} that receive the per-plane CSR."""
    require_cuda(S, weight, weightT, bias, what="spike_linear")
    require_f32(S, bias, what="spike_linear")
    if (weight is None) == (weightT is None):
        raise EngineError("spike_linear: pass exactly one of weight [N, K] or weightT [K, N]")
    squeeze = S.dim() == 2
    S = _contig(S)
    if squeeze:
        S = S.unsqueeze(0)
    if S.dim() != 3:
        raise EngineError(f"spike_linear: S must be [T, M, K] or [M, K], got {tuple(S.shape)}")
    T, M, K = S.shape
    W = weight if weight is not None else weightT
    if W.dtype not in (torch.float32, torch.bfloat16):
        raise EngineError(f"spike_linear: weight dtype {W.dtype} not supported (float32 or bfloat16)")
    if weight is not None:
        N, Kw = weight.shape
        sk, sn = weight.stride(1), weight.stride(0)
    else:
        Kw, N = weightT.shape
        sk, sn = weightT.stride(0), weightT.stride(1)
    if Kw != K:
        raise EngineError(f"spike_linear: weight K={Kw} does not match input K={K}")
    if bias is not None:
        bias = _contig(bias)
        if bias.numel() != N:
            raise EngineError("spike_linear: bias must have N elements")
    wdt = _lib.SPK_BF16 if W.dtype == torch.bfloat16 else _lib.SPK_F32
    lib = _lib.load()
    Y = torch.empty(T, M, N, dtype=torch.float32, device=S.device)
    c = csr or {}
    cap = c["col_idx"].numel() if c else 0
    ws, wsn = _lib.workspace(S.device, lib.spk_spike_linear_workspace_bytes(T, M, K, N, wdt))
    _record("spike_linear", T * M, K, N)
    img = _weight_image(W, K, N, sk, sn, wdt) if _branch(branch) != _lib.BRANCH_CSR else None
    check(lib.spk_spike_linear_img(ptr(S), T, M, K, ptr(W), wdt, sk, sn, N, ptr(img), ptr(bias), ptr(Y),
                                   ptr(c.get("nnz_row")), ptr(c.get("row_ptr")), ptr(c.get("col_idx")),
                                   ptr(c.get("values")), ptr(c.get("plane_ptr")), cap, _branch(branch), ws, wsn,
                                   stream_of(S)), "spk_spike_linear")
    return Y[0] if squeeze else Y


_ACTS = {"none": 0, "heaviside": 1, "vspike": 2, "heaviside_bits": 3, "vspike_bits": 4}


def linear_act(x, weight, bias=None, act="none", thr=0.0):
    """act(x @ weight.T + bias) for x [..., K] fp32 and an nn.Linear weight
    [N, K] fp32 on the tensor cores, fp32-accurate (spk_linear_act):

      "none"       y
      "heaviside"  (y - thr > 0).float()               spike_fn(fc1(x) - thr); q, k spikes (thr 0)
      "vspike"     ((tanh(y) + 1) / 2 - thr > 0).float()  v spikes (thr = tau)
      "heaviside_bits"  the "heaviside" spikes packed 32 to an int32 word:
                   [..., N/32], bit b of word w = column 32w + b (N % 32 == 0)
      "vspike_bits"     the "vspike" spikes packed the same way

    Needs N > 64 and K % 4 == 0."""
    require_cuda(x, weight, bias, what="linear_act")
    require_f32(x, weight, bias, what="linear_act")
    if act not in _ACTS:
        raise EngineError(f"linear_act: act must be one of {sorted(_ACTS)}")
    x = _contig(x)
    K = x.shape[-1]
    N, Kw = weight.shape
    if Kw != K:
        raise EngineError(f"linear_act: weight K={Kw} does not match input K={K}")
    if bias is not None:
        bias = _contig(bias)
        if bias.numel() != N:
            raise EngineError("linear_act: bias must have N elements")
    R = x.numel() // K if K else 0
    if act in ("heaviside_bits", "vspike_bits"):
        if N % 32:
            raise EngineError(f"linear_act: packed spikes need N % 32 == 0 (N={N})")
        Y = torch.empty(*x.shape[:-1], N // 32, dtype=torch.int32, device=x.device)
    else:
        Y = torch.empty(*x.shape[:-1], N, dtype=torch.float32, device=x.device)
    lib = _lib.load()
    ws, wsn = _lib.workspace(x.device, lib.spk_linear_act_workspace_bytes(K, N))
    _record("linear_act", R, K, N)
    img = _weight_image(weight, K, N, weight.stride(1), weight.stride(0), _lib.SPK_F32)
    check(lib.spk_linear_act_img(ptr(x), R, K, ptr(weight), weight.stride(1), weight.stride(0), N, ptr(img),
                                 ptr(bias), _ACTS[act], float(thr), ptr(Y), ws, wsn, stream_of(x)), "spk_linear_act")
    return Y


def engine_linear(lin, x, act="none", thr=0.0):
    """act(lin(x)) through the engine's fp32-accurate tensor-core linear
    (spk_linear_act) when autograd is off and the shape is one it takes
    (out_features > 64, in_features % 4 == 0); None otherwise, and the caller
    runs the module (the reference's own nn.Linear, which training needs)."""
    if torch.is_grad_enabled() or not x.is_cuda or lin.out_features <= 64 or lin.in_features % 4:
        return None
    return linear_act(x, lin.weight, lin.bias, act, thr)


def spike_linear_bits(bits, K, weight, bias=None):
    """Spike-linear over packed spikes: bits int32 [..., K/32] (bit b of word w
    = column 32w + b, as linear_act(act="heaviside_bits") writes them), an
    nn.Linear weight [N, K] fp32, optional bias -> [..., N] fp32; the same
    values as spike_linear(unpack_spikes(bits, K), weight, bias,
    branch="dense").  Needs K % 64 == 0 and N > 64."""
    require_cuda(bits, weight, bias, what="spike_linear_bits")
    require_f32(weight, bias, what="spike_linear_bits")
    if bits.dtype != torch.int32:
        raise EngineError(f"spike_linear_bits: bits must be int32, got {bits.dtype}")
    bits = _contig(bits)
    N, Kw = weight.shape
    if Kw != K or bits.shape[-1] * 32 != K:
        raise EngineError(f"spike_linear_bits: K={K}, weight K={Kw}, bits hold {bits.shape[-1] * 32} columns")
    if bias is not None:
        bias = _contig(bias)
        if bias.numel() != N:
            raise EngineError("spike_linear_bits: bias must have N elements")
    R = bits.numel() // bits.shape[-1]
    Y = torch.empty(*bits.shape[:-1], N, dtype=torch.float32, device=bits.device)
    lib = _lib.load()
    _record("spike_linear_bits", R, K, N)
    img = _weight_image(weight, K, N, weight.stride(1), weight.stride(0), _lib.SPK_F32)
    ws, wsn = (None, 0) if img is not None else _lib.workspace(bits.device, lib.spk_linear_act_workspace_bytes(K, N))
    check(lib.spk_spike_linear_bits(ptr(bits), 1, R, K, ptr(weight), weight.stride(1), weight.stride(0), N, ptr(img),
                                    ptr(bias), ptr(Y), ws, wsn, stream_of(bits)), "spk_spike_linear_bits")
    return Y


def unpack_spikes(bits, K):
    """fp32 0 / 1 spikes [..., K] from packed words [..., K/32] (inspection and
    tests; the engine consumes the packed form directly)."""
    shifts = torch.arange(32, device=bits.device, dtype=torch.int32)
    b = (bits.unsqueeze(-1) >> shifts) & 1
    return b.reshape(*bits.shape[:-1], bits.shape[-1] * 32)[..., :K].float()


def alloc_csr(T, M, K, device, capacity=None, values=False):
    """Preallocated per-plane CSR buffers for spike_linear(csr=...)."""
    cap = int(capacity if capacity is not None else T * M * K)
    d = {
        "nnz_row": torch.empty(T * M, dtype=torch.int32, device=device),
        "row_ptr": torch.empty(T * (M + 1), dtype=torch.int32, device=device),
        "col_idx": torch.empty(max(cap, 1), dtype=torch.int32, device=device),
        "plane_ptr": torch.empty(T + 1, dtype=torch.int64, device=device),
    }
    if values:
        d["values"] = torch.empty(max(cap, 1), dtype=torch.float32, device=device)
    return d


def sparse_multistep_forward(dense_input, weightT, nnz_per_row, row_offsets, col_indices, values, T,
                             branch="auto"):
    """The reference op (sparse_linear.cu:645-691): dense_input [T, B, I],
    weightT [I, O] -> [T, B, O]; the CSR buffers receive plane T-1's CSR."""
    require_cuda(dense_input, weightT, nnz_per_row, row_offsets, col_indices, values,
                 what="sparse_multistep_forward")
    require_f32(dense_input, weightT, values, what="sparse_multistep_forward")
    x = _contig(dense_input)
    T = int(T)
    if x.dim() != 3 or x.shape[0] != T:
        x = x.reshape(T, -1, x.shape[-1])
    _, B, I = x.shape
    wT = _contig(weightT)
    O = wT.shape[1]
    if wT.shape[0] != I:
        raise EngineError(f"sparse_multistep_forward: weightT has {wT.shape[0]} rows, input has {I} features")
    cap = min(col_indices.numel(), values.numel())
    out = torch.empty(T, B, O, dtype=torch.float32, device=x.device)
    lib = _lib.load()
    ws, wsn = _lib.workspace(x.device, lib.spk_sparse_forward_workspace_bytes(T, B, I, O))
    check(lib.spk_sparse_multistep_forward(ptr(x), T, B, I, ptr(wT), O, ptr(nnz_per_row), ptr(row_offsets),
                                           ptr(col_indices), ptr(values), cap, ptr(out), _branch(branch), ws, wsn,
                                           stream_of(x)), "spk_sparse_multistep_forward")
    return out


def sparse_forward(input, weightT, nnz_per_row, row_offsets, col_indices, values, branch="auto"):
    """The reference op (sparse_linear.cu:594-631): input [B, I] -> [B, O]."""
    require_cuda(input, weightT, nnz_per_row, row_offsets, col_indices, values, what="sparse_forward")
    require_f32(input, weightT, values, what="sparse_forward")
    x = _contig(input)
    B, I = x.shape
    wT = _contig(weightT)
    O = wT.shape[1]
    if wT.shape[0] != I:
        raise EngineError(f"sparse_forward: weightT has {wT.shape[0]} rows, input has {I} features")
    cap = min(col_indices.numel(), values.numel())
    out = torch.empty(B, O, dtype=torch.float32, device=x.device)
    lib = _lib.load()
    ws, wsn = _lib.workspace(x.device, lib.spk_sparse_forward_workspace_bytes(1, B, I, O))
    check(lib.spk_sparse_forward(ptr(x), B, I, ptr(wT), O, ptr(nnz_per_row), ptr(row_offsets), ptr(col_indices),
                                 ptr(values), cap, ptr(out), _branch(branch), ws, wsn, stream_of(x)),
          "spk_sparse_forward")
    return out


def dense_to_csr_gpu(dense_input):
    """The reference op dense_to_csr_gpu (sparse_linear.cu:563-588):
    [B, I] -> [row_offsets [B+1], col_indices [B*I], values [B*I]]."""
    require_cuda(dense_input, what="dense_to_csr_gpu")
    require_f32(dense_input, what="dense_to_csr_gpu")
    x = _contig(dense_input)
    B, I = x.shape
    dev = x.device
    row_ptr = torch.empty(B + 1, dtype=torch.int32, device=dev)
    col_idx = torch.empty(B * I, dtype=torch.int32, device=dev)
    vals = torch.empty(B * I, dtype=torch.float32, device=dev)
    plane_ptr = torch.empty(2, dtype=torch.int64, device=dev)
    lib = _lib.load()
    ws, wsn = _lib.workspace(dev, lib.spk_csr_workspace_bytes(1, B, I))
    check(lib.spk_csr_compact(ptr(x), 1, B, I, None, ptr(row_ptr), ptr(col_idx), ptr(vals), ptr(plane_ptr), B * I,
                              ws, wsn, stream_of(x)), "spk_csr_compact")
    return [row_ptr, col_idx, vals]


# ---------------------------------------------------------------------- attention
def apply_channel_decay(k, lam):
    """k_w = k * lam ** (N-1-n) (attention_cuda.cu:42-77)."""
    require_cuda(k, lam, what="apply_channel_decay")
    require_f32(k, lam, what="apply_channel_decay")
    if k.dim() < 2:
        raise EngineError("apply_channel_decay: k must have at least 2 dimensions")
    k = _contig(k)
    lam = _contig(lam)
    d, N = k.shape[-1], k.shape[-2]
    if lam.dim() != 1 or lam.numel() != d:
        raise EngineError("apply_channel_decay: lam must be 1D tensor of size d matching k.size(-1)")
    out = torch.empty_like(k)
    if k.numel() == 0:
        return out
    check(_lib.load().spk_apply_channel_decay(ptr(k), ptr(lam), k.numel() // (N * d), N, d, ptr(out), stream_of(k)),
          "spk_apply_channel_decay")
    return out


def fused_normalize_attention(numer, denom, eps):
    """numer / (denom + eps) elementwise (attention_cuda.cu:79-107)."""
    require_cuda(numer, denom, what="fused_normalize_attention")
    require_f32(numer, denom, what="fused_normalize_attention")
    if denom.numel() < numer.numel():
        raise EngineError("fused_normalize_attention: denom must have at least as many elements as numer")
    numer = _contig(numer)
    denom = _contig(denom)
    out = torch.empty_like(numer)
    check(_lib.load().spk_normalize_attention(ptr(numer), ptr(denom), numer.numel(), float(eps), ptr(out),
                                              stream_of(numer)), "spk_normalize_attention")
    return out


def spiking_attention(q, k, v, lam, heads, eps=1e-6):
    """Fused spiking linear attention: q, k, v spikes [..., L, d] (d = heads*dh)
    -> normalised attention [..., L, d] (the o_proj input of
    AstrocyteHebbianAttention, attention.py:120-135)."""
    require_cuda(q, k, v, lam, what="spiking_attention")
    require_f32(q, k, v, lam, what="spiking_attention")
    shape = q.shape
    L, d = shape[-2], shape[-1]
    if k.shape != shape or v.shape != shape:
        raise EngineError("spiking_attention: q, k and v must have the same shape")
    if d % heads:
        raise EngineError("spiking_attention: d_model must be divisible by heads")
    dh = d // heads
    q, k, v, lam = (_contig(t) for t in (q, k, v, lam))
    BT = q.numel() // (L * d)
    out = torch.empty(shape, dtype=torch.float32, device=q.device)
    lib = _lib.load()
    ws, wsn = _lib.workspace(q.device, lib.spk_attention_workspace_bytes(BT, L, heads, dh))
    check(lib.spk_spiking_attention(ptr(q), ptr(k), ptr(v), ptr(lam), BT, L, heads, dh, float(eps), ptr(out), ws,
                                    wsn, stream_of(q)), "spk_spiking_attention")
    return out


def spiking_attention_bits(q_bits, k_bits, v_bits, lam, heads, eps=1e-6):
    """spiking_attention over packed spikes: q_bits, k_bits, v_bits int32
    [..., L, d/32] (bit b of word w = channel 32w + b, as linear_act's
    "heaviside_bits" / "vspike_bits" write them) -> [..., L, d] fp32, the same
    values as spiking_attention on the unpacked spikes.  Needs d % 128 == 0."""
    require_cuda(q_bits, k_bits, v_bits, lam, what="spiking_attention_bits")
    require_f32(lam, what="spiking_attention_bits")
    shape = q_bits.shape
    if k_bits.shape != shape or v_bits.shape != shape:
        raise EngineError("spiking_attention_bits: q, k and v must have the same shape")
    for t in (q_bits, k_bits, v_bits):
        if t.dtype != torch.int32:
            raise EngineError("spiking_attention_bits: packed spikes must be int32")
    L, d = shape[-2], shape[-1] * 32
    if d % heads:
        raise EngineError("spiking_attention_bits: d_model must be divisible by heads")
    dh = d // heads
    q_bits, k_bits, v_bits, lam = (_contig(t) for t in (q_bits, k_bits, v_bits, lam))
    BT = q_bits.numel() // (L * (d // 32))
    out = torch.empty(*shape[:-1], d, dtype=torch.float32, device=q_bits.device)
    lib = _lib.load()
    ws, wsn = _lib.workspace(q_bits.device, lib.spk_attention_workspace_bytes(BT, L, heads, dh))
    check(lib.spk_spiking_attention_bits(ptr(q_bits), ptr(k_bits), ptr(v_bits), ptr(lam), BT, L, heads, dh,
                                         float(eps), ptr(out), ws, wsn, stream_of(q_bits)),
          "spk_spiking_attention_bits")
    return out


# --------------------------------------------------------------------------- GSMC
def fused_gsmc_step(gi, gr, wd, bias, m, s, heat, v_th, gate_scale, adaptive_threshold, beta_adapt):
    """One GSMC step (gsmc_cuda.cu:79-127); updates m, s, heat in place and
    returns the new spikes [M, d]."""
    require_cuda(gi, gr, wd, bias, m, s, heat, what="fused_gsmc_step")
    require_f32(gi, gr, wd, bias, m, s, heat, what="fused_gsmc_step")
    for t in (gi, gr, wd, bias, m, s, heat):
        if not t.is_contiguous():
            raise EngineError("fused_gsmc_step: inputs and state tensors must be contiguous")
    M, d = gi.shape[0], wd.shape[-1]
    if gi.shape[-1] != 4 * d or gr.shape[-1] != 4 * d:
        raise EngineError("fused_gsmc_step: gi and gr must be of shape (M, 4*d)")
    if bias.numel() != 4 * d:
        raise EngineError("fused_gsmc_step: bias must have 4*d elements")
    if m.numel() != M * d or s.numel() != M * d or heat.numel() != M * d:
        raise EngineError("fused_gsmc_step: m, s and heat must be of size (M, d)")
    out = torch.empty(M, d, dtype=torch.float32, device=gi.device)
    check(_lib.load().spk_gsmc_step(ptr(gi), ptr(gr), ptr(wd), ptr(bias), ptr(m), ptr(s), ptr(heat), ptr(out), M, d,
                                    float(v_th), float(gate_scale), int(bool(adaptive_threshold)),
                                    float(beta_adapt), stream_of(gi)), "spk_gsmc_step")
    return out


def gsmc_forward(gi_all, wd_all, w_rec, bias, v_th=1.0, gate_scale=4.0, adaptive=True, beta=0.8, pool="mean",
                 return_planes=False, fused=False):
    """The eval-mode GSMC recurrence (gsmc.py:96-148) over precomputed input
    projections gi_all [T, M, 4d] and wd_all [T, M, d]; w_rec is the W_rec
    nn.Linear weight [4d, d].  Returns pooled [M, d] (and the planes [T, M, d]).
    fused=True: the recurrent projection and the cell update in one kernel per
    plane (SPK_GSMC_FUSED; same results, slower at the model's geometry)."""
    require_cuda(gi_all, wd_all, w_rec, bias, what="gsmc_forward")
    require_f32(gi_all, wd_all, w_rec, bias, what="gsmc_forward")
    gi_all, wd_all, w_rec, bias = (_contig(t) for t in (gi_all, wd_all, w_rec, bias))
    T, M, d = wd_all.shape
    pooled = torch.empty(M, d, dtype=torch.float32, device=gi_all.device)
    planes = torch.empty(T, M, d, dtype=torch.float32, device=gi_all.device) if return_planes else None
    lib = _lib.load()
    ws, wsn = _lib.workspace(gi_all.device, lib.spk_gsmc_workspace_bytes(M, d))
    _record("gsmc_recurrent", (T - 1) * M, d, 4 * d)  # W_rec s_{t-1} for t >= 1 (s_{-1} = 0 is skipped)
    check(lib.spk_gsmc_forward_ex(ptr(gi_all), ptr(wd_all), ptr(w_rec), ptr(bias), T, M, d, float(v_th),
                                  float(gate_scale), int(bool(adaptive)), float(beta), 1 if pool == "mean" else 0,
                                  ptr(planes), ptr(pooled), ws, wsn, 1 if fused else 0, stream_of(gi_all)),
          "spk_gsmc_forward")
    return (pooled, planes) if return_planes else pooled


# --------------------------------------------------------------------------- residual add + layer norm
def add_layernorm(x, delta, weight=None, bias=None, eps=1e-5):
    """h = x + delta and y = layer_norm(h) over the last dimension in one pass
    (spk_add_layernorm): the pre-norm block's residual add followed by the
    nn.LayerNorm of the sum (nn/attention.py:174-177).  delta None: h = x and
    y = layer_norm(x).  weight / bias: the nn.LayerNorm affine parameters [d]
    (None: 1 / 0).  Returns (h, y).  Needs d % 4 == 0 and d <= 1024."""
    require_cuda(x, delta, weight, bias, what="add_layernorm")
    require_f32(x, delta, weight, bias, what="add_layernorm")
    x = _contig(x)
    d = x.shape[-1]
    if delta is not None:
        if delta.shape != x.shape:
            raise EngineError(f"add_layernorm: delta shape {tuple(delta.shape)} != x shape {tuple(x.shape)}")
        delta = _contig(delta)
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and p.numel() != d:
            raise EngineError(f"add_layernorm: {name} must have d={d} elements")
    weight = _contig(weight) if weight is not None else None
    bias = _contig(bias) if bias is not None else None
    rows = x.numel() // d if d else 0
    h = torch.empty_like(x) if delta is not None else x
    y = torch.empty_like(x)
    check(_lib.load().spk_add_layernorm(ptr(x), ptr(delta), ptr(weight), ptr(bias), rows, d, float(eps),
                                        ptr(h) if delta is not None else None, ptr(y), stream_of(x)),
          "spk_add_layernorm")
    return h, y


# --------------------------------------------------------------------------- Spire planes
def spire_planes(u, dither, frontier=None, temporal_frontier=None):
    """The Spire encoder's temporal planes (encode/spire.py:60-69) in one pass
    (spk_spire_planes): for u [B, N, d] and dither [T],
    planes[t] = ((u - frontier) - temporal_frontier[n]) - dither[t] > 0 as
    float32 [T, B, N, d]; frontier [d] and temporal_frontier [N] (any shape
    with those element counts) may be None."""
    require_cuda(u, dither, frontier, temporal_frontier, what="spire_planes")
    require_f32(u, dither, frontier, temporal_frontier, what="spire_planes")
    if u.dim() != 3:
        raise EngineError("spire_planes: u must be (B, N, d)")
    B, N, d = u.shape
    u = _contig(u)
    dither = _contig(dither).view(-1)
    if frontier is not None:
        frontier = _contig(frontier).view(-1)
        if frontier.numel() != d:
            raise EngineError(f"spire_planes: frontier must have d={d} elements")
    if temporal_frontier is not None:
        temporal_frontier = _contig(temporal_frontier).view(-1)
        if temporal_frontier.numel() != N:
            raise EngineError(f"spire_planes: temporal_frontier must have N={N} elements")
    T = dither.numel()
    planes = torch.empty(T, B, N, d, dtype=torch.float32, device=u.device)
    check(_lib.load().spk_spire_planes(ptr(u), ptr(frontier), ptr(temporal_frontier), ptr(dither), T, B, N, d,
                                       ptr(planes), stream_of(u)), "spk_spire_planes")
    return planes


def spire_dither(v, dither):
    """spire_dither(v [B, N, d], dither [T]) -> (v - dither[t] > 0) as float32
    [T, B, N, d]: the reference Spire engine's entry point (spire_cuda.cu:28-58)."""
    return spire_planes(v, dither)


# --------------------------------------------------------------------------- readout pooling
def temporal_mean(x):
    """(mean of x, mean of (x > 0)) over (t, n) per sample and channel for a
    temporal context x [T, B, N, d], or over n for [B, N, d] (the pooling in
    front of SpikingTransformer's classifier, models/transformer.py:159-192),
    in one pass (spk_temporal_mean).  Both results [B, d] float32."""
    require_cuda(x, what="temporal_mean")
    require_f32(x, what="temporal_mean")
    if x.dim() == 3:
        T, (B, N, d) = 1, x.shape
    elif x.dim() == 4:
        T, B, N, d = x.shape
    else:
        raise EngineError("temporal_mean: x must be (T, B, N, d) or (B, N, d)")
    x = _contig(x)
    mean_x = torch.empty(B, d, dtype=torch.float32, device=x.device)
    mean_s = torch.empty(B, d, dtype=torch.float32, device=x.device)
    check(_lib.load().spk_temporal_mean(ptr(x), T, B, N, d, ptr(mean_x), ptr(mean_s), stream_of(x)),
          "spk_temporal_mean")
    return mean_x, mean_s


# --------------------------------------------------------------------------- training and streaming operators
# The operators below take float32, bfloat16 or float16 tensors (fp32
# arithmetic, results rounded once) and are differentiable.  Scratch memory is
# allocated per call, so calls on several streams and captured graphs never
# share any.
_DTYPES = {torch.float32: _lib.SPK_F32, torch.bfloat16: _lib.SPK_BF16, torch.float16: _lib.SPK_F16}


def _checked(what, x, *others):
    """The dtype code of x, a CUDA tensor of one of the three types; the others
    (or None) on its device."""
    try:
        dev = x.get_device() if x.is_cuda else -1
        same = dev >= 0
        for t in others:
            if t is not None and t.get_device() != dev:
                same = False
    except AttributeError:
        same = False
    if not same:
        require_cuda(x, *others, what=what)
        if x is None:
            raise EngineError(f"{what}: CUDA tensors required (this engine has no CPU path)")
        raise EngineError(f"{what}: tensors on several devices")
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise EngineError(f"{what}: float32, bfloat16 or float16 tensors required, got {x.dtype}")
    return code


_ENTRY = {}


def _call(t, name, *args):
    """Entry point `name` on t's device and its current stream (the last argument)."""
    fn = _ENTRY.get(name)
    if fn is None:
        fn = _ENTRY[name] = getattr(_lib.load(), name)
    dev = t.get_device()
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc, name)


def _scratch(t, nbytes):
    return t.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _backward(fn):
    """A Function's backward made of engine calls, which have no backward of
    their own: differentiating it again raises (and only then costs the wrapper)."""
    guarded = torch.autograd.function.once_differentiable(fn)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return staticmethod(backward)


# ------------------------------------------------------------- gated linear recurrence
_FORMS = {"gate": 0, "leaky": 1}


def _form(form, what):
    try:
        return _FORMS[form]
    except (KeyError, TypeError):
        raise EngineError(f"{what}: form must be one of {sorted(_FORMS)}, got {form!r}") from None


@functools.lru_cache(maxsize=1024)
def _flat_strides(shape, strides, dim):
    if shape[-1] > 1 and strides[-1] != 1:
        return None
    step, size = None, 1
    for i in range(len(shape) - 2, -1, -1):  # from the innermost batch dimension outwards
        n = shape[i]
        if i == dim or n == 1:
            continue
        if step is None:
            step, size = strides[i], n
        elif strides[i] != step * size:
            return None
        else:
            size *= n
    return (step if step is not None else 0), strides[dim]


def _time_strides(t, dim):
    """(stride of the flattened batch, stride of time) of t with time at
    dimension `dim` and every other dimension but the last one batch; None when
    the batch dimensions do not flatten or the last one is not contiguous."""
    return _flat_strides(t.shape, t.stride(), dim)


def _time_major(t, dim):
    """t itself, or a copy whose batch dimensions flatten, and its _time_strides."""
    st = _time_strides(t, dim)
    if st is not None:
        return t, st
    t = t.movedim(dim, -2).contiguous().movedim(-2, dim)
    return t, _time_strides(t, dim)


def _empty_time(t, dim):
    """An uninitialised tensor of t's shape whose batch dimensions flatten, and its strides."""
    out = torch.empty_like(t, memory_format=torch.contiguous_format)
    st = _time_strides(out, dim)
    if st is None:  # time between the batch dimensions: laid out behind them
        shape = list(t.shape)
        steps = shape.pop(dim)
        shape.insert(len(shape) - 1, steps)
        out = t.new_empty(shape).movedim(-2, dim)
        st = _time_strides(out, dim)
    return out, st


def _recurrence_forward(x, gate, state, form, dim, lengths, keep):
    """(h, last, carry) through spk_recurrence; `keep`: fill carry for the backward pass."""
    lib = _lib.load()
    L, D = x.shape[dim], x.shape[-1]
    B = x.numel() // (L * D) if x.numel() else (state.numel() // D if D else 0)
    (x, (xb, xt)), (gate, (gb, gt)), (h, (hb, ht)) = _time_major(x, dim), _time_major(gate, dim), _empty_time(x, dim)
    last = torch.empty_like(state)
    carry = None
    if keep:
        chunk = int(lib.spk_recurrence_chunk(_DTYPES[x.dtype], B, L, D))
        if L > chunk:
            carry = x.new_empty((L + chunk - 1) // chunk - 1, B, D, dtype=torch.float32)
    _call(x, "spk_recurrence", ptr(x), xb, xt, ptr(gate), gb, gt, _DTYPES[x.dtype], form, B, L, D, ptr(state),
          ptr(lengths), ptr(h), hb, ht, ptr(last), ptr(carry))
    return h, last, carry


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, form, dim, lengths):
        h, last, carry = _recurrence_forward(x, gate, state, form, dim, lengths, True)
        ctx.save_for_backward(x, gate, state, lengths, carry)
        ctx.form, ctx.dim = form, dim
        ctx.set_materialize_grads(False)
        return h, last

    @_backward
    def backward(ctx, gh, glast):
        x, gate, state, lengths, carry = ctx.saved_tensors
        if gh is None and glast is None:
            return (None,) * 6
        dim = ctx.dim
        L, D = x.shape[dim], x.shape[-1]
        B = state.numel() // D if D else 0
        (x, (xb, xt)), (gate, (gb, gt)) = _time_major(x, dim), _time_major(gate, dim)
        ghb = ght = 0
        if gh is not None:
            gh, (ghb, ght) = _time_major(gh, dim)
        glast = None if glast is None else _contig(glast)
        dx, (db, dt) = _empty_time(x, dim)
        dgate = torch.empty_like(dx)  # dense: the same strides
        dstate = torch.empty_like(state)
        _call(x, "spk_recurrence_backward", ptr(x), xb, xt, ptr(gate), gb, gt, ptr(gh), ghb, ght, _DTYPES[x.dtype],
              ctx.form, B, L, D, ptr(state), ptr(lengths), ptr(carry), ptr(glast), ptr(dx), ptr(dgate), db, dt,
              ptr(dstate))
        return dx, dgate, dstate, None, None, None


def gated_recurrence(x, gate, state=None, form="leaky", dim=-2, lengths=None):
    """Gated linear recurrence along dimension `dim` of x [..., d] (any but the
    last), with gate of x's shape and dtype (spk_recurrence):

      "leaky"  h_t = a_t h_{t-1} + (1 - a_t) x_t,  a_t = sigmoid(gate_t)
      "gate"   h_t = gate_t h_{t-1} + x_t

    from `state` (float32, x's shape without `dim`; None: zero).  Returns (h,
    last): h like x, last the float32 state after the last step, to be handed
    to the next call or to gated_recurrence_step.  ``lengths`` (int32 or int64,
    x's shape without `dim` and the last dimension; clamped to [0, steps]):
    steps at or beyond a row's length are not read, h is 0 there and the state
    stays.  x and gate may be slices or broadcast views whose last dimension is
    contiguous.  Differentiable in x, gate and state."""
    what = "gated_recurrence"
    _checked(what, x, gate, state, lengths)
    form = _form(form, what)
    if gate.dtype != x.dtype or gate.shape != x.shape:
        raise EngineError(f"{what}: gate must have x's shape and dtype ({tuple(x.shape)}, {x.dtype}), "
                          f"got {tuple(gate.shape)}, {gate.dtype}")
    if x.dim() < 2 or not -x.dim() <= dim < x.dim() or dim % x.dim() == x.dim() - 1:
        raise EngineError(f"{what}: dim must name a dimension of x but the last, got {dim} for {tuple(x.shape)}")
    dim %= x.dim()
    shape = x.shape[:dim] + x.shape[dim + 1:]
    if state is None:
        state = x.new_zeros(shape, dtype=torch.float32)
    elif state.dtype != torch.float32 or state.shape != shape:
        raise EngineError(f"{what}: state must be float32 of shape {tuple(shape)}, got {tuple(state.shape)}, "
                          f"{state.dtype}")
    if lengths is not None:
        if lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != shape[:-1]:
            raise EngineError(f"{what}: lengths must be int32 or int64 of shape {tuple(shape[:-1])}, got "
                              f"{tuple(lengths.shape)}, {lengths.dtype}")
        if lengths.dtype == torch.int64:  # clamped first: the cast wraps
            lengths = lengths.clamp(0, x.shape[dim]).to(torch.int32)
        lengths = _contig(lengths)
    state = _contig(state)
    if _wants_grad(x, gate, state):
        return _GatedRecurrence.apply(x, gate, state, form, dim, lengths)
    return _recurrence_forward(x, gate, state, form, dim, lengths, False)[:2]


def _rows(t):
    """t, or a contiguous copy, as rows of its last dimension, and their stride."""
    if t.is_contiguous():
        return t, t.shape[-1]
    st = _time_strides(t.unsqueeze(-2), t.dim() - 1)  # a time dimension of one step: the batch is the rows
    return (t, st[0]) if st is not None else (t.contiguous(), t.shape[-1])


def gated_recurrence_step(x, gate, state, form="leaky", new_state=None):
    """One step of gated_recurrence for streaming: x and gate [..., d] of one
    time step, state float32 of the same shape -> (h, new state): h in x's
    dtype, the state in float32.  ``new_state``: the tensor to write it to
    (contiguous float32; `state` itself updates it in place).  x and gate may be
    slices whose last dimension is contiguous.  Not differentiable."""
    what = "gated_recurrence_step"
    # one chain of cheap tests for the call that is right (a stream makes it per
    # plane); what is wrong is looked for only when it fails
    try:
        shape = x.shape
        dt, fm, dev = _DTYPES[x.dtype], _FORMS[form], x.get_device()
        right = (dev >= 0 and gate.dtype == x.dtype and gate.shape == shape and gate.get_device() == dev
                 and state.dtype == torch.float32 and state.shape == shape and state.get_device() == dev
                 and (new_state is None or (new_state.dtype == torch.float32 and new_state.shape == shape
                                            and new_state.get_device() == dev and new_state.is_contiguous()))
                 and len(shape) > 0 and not _wants_grad(x, gate, state))
    except (AttributeError, KeyError, TypeError):
        right = False
    if not right:
        _checked(what, x, gate, state, new_state)
        _form(form, what)
        if gate.dtype != x.dtype or gate.shape != x.shape:
            raise EngineError(f"{what}: gate must have x's shape and dtype")
        if state.dtype != torch.float32 or state.shape != x.shape:
            raise EngineError(f"{what}: state must be float32 of x's shape {tuple(x.shape)}")
        if _wants_grad(x, gate, state):
            raise EngineError(f"{what}: no backward pass (use gated_recurrence, or torch.no_grad())")
        if not x.shape:
            raise EngineError(f"{what}: x must have a channel dimension")
        raise EngineError(f"{what}: new_state must be contiguous float32 of x's shape {tuple(x.shape)}")
    D = shape[-1]
    if x.is_contiguous():
        out, xs = torch.empty_like(x), D
    else:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        x, xs = _rows(x)
    gate, gs = (gate, D) if gate.is_contiguous() else _rows(gate)
    state = _contig(state)
    if new_state is None:
        new_state = torch.empty_like(state)
    _call(x, "spk_recurrence_step", x.data_ptr(), xs, gate.data_ptr(), gs, dt, fm, out.numel() // D if D else 0, D,
          state.data_ptr(), out.data_ptr(), new_state.data_ptr())
    return out, new_state


# ------------------------------------------------------------- group norm + activation
_NORM_ACTS = {"none": 0, "heaviside": 1, "silu": 5}


def _group_norm_forward(x, groups, weight, bias, eps, act, thr, keep):
    """(y, mean, rstd) through spk_group_norm_act; mean and rstd [S, G] when `keep`."""
    lib = _lib.load()
    S, C = x.shape[0], x.shape[-1]
    P = x.numel() // (S * C) if S else 0
    y = torch.empty_like(x)
    mean, rstd = x.new_empty(2, S, groups, dtype=torch.float32) if keep else (None, None)
    ws = _scratch(x, lib.spk_group_norm_workspace_bytes(_DTYPES[x.dtype], S, P, C, groups))
    _call(x, "spk_group_norm_act", ptr(x), _DTYPES[x.dtype], S, P, C, groups, ptr(weight), ptr(bias), eps, act, thr,
          ptr(y), ptr(mean), ptr(rstd), ptr(ws), 0 if ws is None else ws.numel())
    return y, mean, rstd


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, thr):
        y, mean, rstd = _group_norm_forward(x, groups, weight, bias, eps, act, thr, True)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.groups, ctx.act, ctx.thr = groups, act, thr
        return y

    @_backward
    def backward(ctx, gy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        lib = _lib.load()
        gy = _contig(gy)
        S, C = x.shape[0], x.shape[-1]
        P = x.numel() // (S * C) if S else 0
        dx = torch.empty_like(x)
        dweight = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        dbias = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        ws = _scratch(x, lib.spk_group_norm_workspace_bytes(_DTYPES[x.dtype], S, P, C, ctx.groups))
        _call(x, "spk_group_norm_act_backward", ptr(x), ptr(gy), _DTYPES[x.dtype], S, P, C, ctx.groups, ptr(weight),
              ptr(bias), ptr(mean), ptr(rstd), ctx.act, ctx.thr, ptr(dx), ptr(dweight), ptr(dbias), ptr(ws),
              0 if ws is None else ws.numel())
        return dx, dweight, dbias, None, None, None, None


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="none", thr=0.0):
    """act(group norm of x) for channels-last x [S, ..., C] (spk_group_norm_act):
    per sample (the first dimension) and group of C / groups neighbouring
    channels, normalised over all positions in between, then scaled by weight
    [C] and shifted by bias [C] (float32; None: 1 / 0), then

      "none"       z
      "silu"       z sigmoid(z)
      "heaviside"  (z - thr > 0), with spike_fn's surrogate gradient

    A (T, B, N, d) tensor is normalised per time plane and sample as
    x.flatten(0, 1).  Differentiable in x, weight and bias."""
    what = "group_norm_act"
    _checked(what, x, weight, bias)
    require_f32(weight, bias, what=what)
    if act not in _NORM_ACTS:
        raise EngineError(f"{what}: act must be one of {sorted(_NORM_ACTS)}")
    if x.dim() < 2 or x.shape[-1] == 0:
        raise EngineError(f"{what}: x must be (samples, ..., channels), got {tuple(x.shape)}")
    C, groups = x.shape[-1], int(groups)
    if groups < 1 or C % groups:
        raise EngineError(f"{what}: {C} channels do not form {groups} groups")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and p.shape != (C,):
            raise EngineError(f"{what}: {name} must have shape ({C},), got {tuple(p.shape)}")
    x = _contig(x)
    weight = None if weight is None else _contig(weight)
    bias = None if bias is None else _contig(bias)
    if _wants_grad(x, weight, bias):
        return _GroupNormAct.apply(x, weight, bias, groups, float(eps), _NORM_ACTS[act], float(thr))
    return _group_norm_forward(x, groups, weight, bias, float(eps), _NORM_ACTS[act], float(thr), False)[0]


# ------------------------------------------------------------- dropout
def _dropout_call(x, residual, p, key):
    y = torch.empty_like(x)
    dev = key if isinstance(key, torch.Tensor) else None
    seed, offset = (0, 0) if dev is not None else key
    _call(x, "spk_dropout", ptr(x), ptr(residual), _DTYPES[x.dtype], x.numel(), p, seed, offset, ptr(dev), ptr(y))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, key):
        ctx.p = p
        ctx.key = None if isinstance(key, torch.Tensor) else key
        ctx.save_for_backward(key if ctx.key is None else None)
        return _dropout_call(x, residual, p, key)

    @_backward
    def backward(ctx, gy):
        key = ctx.saved_tensors[0] if ctx.key is None else ctx.key
        gx = _dropout_call(_contig(gy), None, ctx.p, key) if ctx.needs_input_grad[0] else None
        return gx, (gy if ctx.needs_input_grad[1] else None), None, None


def dropout(x, p, key, residual=None):
    """Dropout with the residual added: residual + keep * x / (1 - p)
    (spk_dropout).  The mask is a function of `key` = (seed, offset) and the
    element's index in x -- a counter-based generator -- and is never stored:
    the backward pass makes it again.  ``key``: two Python integers, or an
    int64 CUDA tensor of two elements, read by the kernel, so that a captured
    graph takes new numbers when the tensor is changed (it must keep its value
    from the forward to the backward pass).  Give every call of a step its own
    offset.  Differentiable in x and residual."""
    what = "dropout"
    _checked(what, x, residual)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise EngineError(f"{what}: p must lie in [0, 1], got {p}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise EngineError(f"{what}: residual must have x's shape and dtype ({tuple(x.shape)}, {x.dtype}), "
                          f"got {tuple(residual.shape)}, {residual.dtype}")
    if isinstance(key, torch.Tensor):
        _checked(what, x, key)
        if key.dtype != torch.int64 or key.shape != (2,):
            raise EngineError(f"{what}: key must be int64 of shape (2,), got {tuple(key.shape)}, {key.dtype}")
        key = _contig(key)
    else:
        try:
            seed, offset = (int(v) & 0xFFFFFFFFFFFFFFFF for v in key)
        except (TypeError, ValueError):
            raise EngineError(f"{what}: key must be two integers or an int64 CUDA tensor") from None
        key = (seed, offset)
    x = _contig(x)
    residual = None if residual is None else _contig(residual)
    if _wants_grad(x, residual):
        return _Dropout.apply(x, residual, p, key)
    return _dropout_call(x, residual, p, key)
