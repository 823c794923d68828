"""torch-tensor front end of the C ABI (device memory and streams come from
torch; all arithmetic runs in libmc_hip.so's HIP kernels).

Shapes follow the reference: x [..., K], W [N, K], A [K, r], B [r, N]; the
leading dims of x are folded into T tokens as FusedLoRAOp::extract_dimensions
does (src/backend/custom_ops.rs:254-270). Activations are float32 or bfloat16;
A, B and their gradients are float32. Every call enqueues on torch's current
stream of the tensors' device and does not synchronise.
"""
import array
import ctypes
import itertools
import operator

import torch

from . import _lib
from ._lib import (AdamWConfig, AdamWTensor, AttnDesc, DistillDesc, EmbeddingDesc, LogprobDesc, LoraDesc, LoraProj,
                   McError, PackedAttnDesc, PolicyDesc, PreferenceDesc, XentDesc, check, lib)

_DTYPES = {torch.float32: _lib.MC_F32, torch.bfloat16: _lib.MC_BF16}
_DTYPE_OF = operator.attrgetter("dtype")


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(t):
    # The raw handle (0.1 us) and not a Stream object around it (1.9 us of a
    # 15 us decode call); current_stream refuses what is not on a GPU.
    if t.is_cuda:
        return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(t.get_device()))
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _dtype_code(t):
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise McError(_lib.MC_ERR_DTYPE, f"unsupported dtype {t.dtype} (float32 or bfloat16)")


def _contig(t, name):
    if t is None:
        return None
    if not t.is_contiguous():
        raise McError(_lib.MC_ERR_LAYOUT, f"{name} must be contiguous")
    return t


def _expect(t, name, shape=None, dtype=None, device=None):
    """Raise McError unless t is contiguous with the given shape, dtype and
    device. These checks run before the C ABI is called: the kernels read
    each buffer over the extent its shape arguments give, so a tensor of the
    wrong size must never reach them."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise McError(_lib.MC_ERR_NULL, f"{name} must be a tensor")
    _contig(t, name)
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise McError(_lib.MC_ERR_SHAPE, f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise McError(_lib.MC_ERR_DTYPE, f"{name} has dtype {t.dtype}, expected {dtype}")
    if device is not None and t.device != device:
        raise McError(_lib.MC_ERR_LAYOUT, f"{name} is on {t.device}, expected {device}")
    return t


def _lora_factors(A, B):
    """FusedLoRAOp::new (src/backend/custom_ops.rs:118-148): A [K, r] and B [r, N]."""
    for t, n in ((A, "A"), (B, "B")):
        if not isinstance(t, torch.Tensor):
            raise McError(_lib.MC_ERR_NULL, f"{n} must be a tensor")
    if A.dim() != 2 or B.dim() != 2:
        raise McError(_lib.MC_ERR_SHAPE,
                      f"LoRA matrices must be 2D, got shapes {list(A.shape)} and {list(B.shape)}")
    if A.shape[1] != B.shape[0]:
        raise McError(_lib.MC_ERR_SHAPE, "Incompatible LoRA matrix dimensions: "
                      f"{A.shape[0]}\u00d7{A.shape[1]} and {B.shape[0]}\u00d7{B.shape[1]}")
    return A.shape[0], A.shape[1], B.shape[1]


def _rows_of(x, name):
    if not isinstance(x, torch.Tensor):
        raise McError(_lib.MC_ERR_NULL, f"{name} must be a tensor")
    if x.dim() < 1:
        raise McError(_lib.MC_ERR_SHAPE, "Input must have at least 1 dimension")
    _contig(x, name)
    _dtype_code(x)
    D = x.shape[-1]
    return (x.numel() // D if D else 0), D


def _workspace(nbytes, device):
    if nbytes == 0:
        return None
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def lora_desc(tokens, in_features, out_features, rank, scale, dropout_p=0.0, dtype=torch.bfloat16):
    return LoraDesc(tokens, in_features, out_features, rank, scale, dropout_p, _DTYPES[dtype])


def lora_forward(x, A, B, scale, W=None, bias=None, mask=None, dropout_p=0.0, save_hidden=True):
    """y = x.W^T + bias + scale*((x.A) (.) mask/(1-p)).B ; returns (y, h_save).

    x [..., K] (float32 or bfloat16), A [K, r] and B [r, N] float32, W [N, K]
    and bias [N] in x's dtype, mask uint8 [T, r] (T = the leading dims of x
    folded); all contiguous on x's device. Shape errors keep the reference's
    messages (custom_ops.rs:123-139, 153-174)."""
    K, r, N = _lora_factors(A, B)
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise McError(_lib.MC_ERR_SHAPE, "Input must have at least 1 dimension")
    _contig(x, "x")
    code = _dtype_code(x)
    if x.shape[-1] != K:
        raise McError(_lib.MC_ERR_SHAPE, f"Input feature dimension mismatch: expected {K}, got {x.shape[-1]}")
    T = x.numel() // K if K else 0
    dev = x.device
    _expect(A, "A", dtype=torch.float32, device=dev)
    _expect(B, "B", dtype=torch.float32, device=dev)
    _expect(W, "W", shape=(N, K), dtype=x.dtype, device=dev)
    _expect(bias, "bias", shape=(N,), dtype=x.dtype, device=dev)
    _expect(mask, "mask", shape=(T, r), dtype=torch.uint8, device=dev)
    d = LoraDesc(T, K, N, r, float(scale), float(dropout_p), code)
    y = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=dev)
    h = torch.empty(r, T, dtype=torch.float32, device=dev) if save_hidden else None
    ws_n = lib().mc_lora_fwd_workspace_size(ctypes.byref(d))  # 0 for an invalid descriptor
    ws = _workspace(ws_n, dev)
    check(lib().mc_lora_fwd(ctypes.byref(d), _ptr(x), _ptr(W), _ptr(bias), _ptr(A), _ptr(B), _ptr(mask),
                            _ptr(y), _ptr(h), _ptr(ws), ws_n, _stream(x)))
    return y, h


def lora_backward(x, A, B, dY, scale, W=None, mask=None, dropout_p=0.0, h_save=None,
                  need_dx=True, need_dA=True, need_dB=True):
    """(dX, dA, dB) with W frozen; entries not requested are None.

    dY [..., N] with x [..., K] over the same leading dims (x may be None
    when dA is not requested), h_save [r, T] float32 from lora_forward
    (required for dB), other tensors as in lora_forward."""
    K, r, N = _lora_factors(A, B)
    if not isinstance(dY, torch.Tensor) or dY.dim() < 1:
        raise McError(_lib.MC_ERR_SHAPE, "dY must have at least 1 dimension")
    _contig(dY, "dY")
    code = _dtype_code(dY)
    if dY.shape[-1] != N:
        raise McError(_lib.MC_ERR_SHAPE, f"dY feature dimension mismatch: expected {N}, got {dY.shape[-1]}")
    T = dY.numel() // N if N else 0
    dev = dY.device
    _expect(A, "A", dtype=torch.float32, device=dev)
    _expect(B, "B", dtype=torch.float32, device=dev)
    _expect(x, "x", shape=tuple(dY.shape[:-1]) + (K,), dtype=dY.dtype, device=dev)
    _expect(W, "W", shape=(N, K), dtype=dY.dtype, device=dev)
    _expect(mask, "mask", shape=(T, r), dtype=torch.uint8, device=dev)
    _expect(h_save, "h_save", shape=(r, T), dtype=torch.float32, device=dev)
    d = LoraDesc(T, K, N, r, float(scale), float(dropout_p), code)
    dX = torch.empty(*dY.shape[:-1], K, dtype=dY.dtype, device=dev) if need_dx else None
    dA = torch.empty(K, r, dtype=torch.float32, device=dev) if need_dA else None
    dB = torch.empty(r, N, dtype=torch.float32, device=dev) if need_dB else None
    ws_n = lib().mc_lora_bwd_workspace_size(ctypes.byref(d))  # 0 for an invalid descriptor
    ws = _workspace(ws_n, dev)
    check(lib().mc_lora_bwd(ctypes.byref(d), _ptr(x), _ptr(W), _ptr(A), _ptr(B), _ptr(mask), _ptr(h_save),
                            _ptr(dY), _ptr(dX), _ptr(dA), _ptr(dB), _ptr(ws), ws_n, _stream(dY)))
    return dX, dA, dB


def _ptr_array(ts):
    return (ctypes.c_void_p * len(ts))(*[None if t is None else t.data_ptr() for t in ts])


def _group_table(x, projs, dropout_p, lead=None, like=None):
    """Validate a grouped call's projections (dicts with W, bias, A, B, mask)
    against the shared x [..., K] and build the C table; returns (table, K,
    r, T, [N_g]). With x None, the leading dims come from `lead`, K from the
    first projection's A and the dtype / device from the tensor `like`."""
    if not isinstance(projs, (list, tuple)) or not 1 <= len(projs) <= _lib.MC_LORA_MAX_GROUP:
        raise McError(_lib.MC_ERR_SHAPE, f"a group holds 1 to {_lib.MC_LORA_MAX_GROUP} projections")
    if x is None:
        if not isinstance(projs[0], dict) or not isinstance(projs[0].get("A"), torch.Tensor) or projs[0]["A"].dim() != 2:
            raise McError(_lib.MC_ERR_SHAPE, "lora_a must be 2D")
        K = projs[0]["A"].shape[0]
        T = 1
        for n in lead:
            T *= n
        dtype, device = like.dtype, like.device
    else:
        if not isinstance(x, torch.Tensor) or x.dim() < 1:
            raise McError(_lib.MC_ERR_SHAPE, "Input must have at least 1 dimension")
        _contig(x, "x")
        K = x.shape[-1]
        T = x.numel() // K if K else 0
        dtype, device = x.dtype, x.device
    if dtype != torch.bfloat16:
        raise McError(_lib.MC_ERR_DTYPE, "grouped projections run in bfloat16 only")
    table = (LoraProj * len(projs))()
    r0, Ns = None, []
    for g, p in enumerate(projs):
        Kg, r, N = _lora_factors(p["A"], p["B"])
        if Kg != K:
            raise McError(_lib.MC_ERR_SHAPE, f"Input feature dimension mismatch: expected {Kg}, got {K}")
        if r0 is not None and r != r0:
            raise McError(_lib.MC_ERR_SHAPE, f"projection {g}: rank {r} differs from the group's {r0}")
        r0 = r
        _expect(p["A"], "A", dtype=torch.float32, device=device)
        _expect(p["B"], "B", dtype=torch.float32, device=device)
        _expect(p.get("W"), "W", shape=(N, K), dtype=dtype, device=device)
        _expect(p.get("bias"), "bias", shape=(N,), dtype=dtype, device=device)
        _expect(p.get("mask"), "mask", shape=(T, r), dtype=torch.uint8, device=device)
        _expect(p.get("Wt"), "Wt", shape=(K, N), dtype=dtype, device=device)
        table[g] = LoraProj(N, *[None if p.get(k) is None else p[k].data_ptr()
                                 for k in ("W", "bias", "A", "B", "mask", "Wt")])
        Ns.append(N)
    return table, K, r0, T, Ns


def lora_group_forward(x, projs, scale, dropout_p=0.0, save_hidden=True):
    """The LoRA projections of one input x [..., K] in one call
    (mc_lora_group_fwd): projs is a list of 1-4 dicts with W [N_g, K], bias
    [N_g] (or None), A [K, r], B [r, N_g], mask [T, r] (or None) and,
    optionally, Wt = transpose_weight(W) for the backward. Returns ([y_g],
    [h_save_g]); each y_g equals lora_forward's for that projection."""
    table, K, r, T, Ns = _group_table(x, projs, dropout_p)
    d = LoraDesc(T, K, Ns[0], r, float(scale), float(dropout_p), _lib.MC_BF16)
    ys = [torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=x.device) for N in Ns]
    hs = [torch.empty(r, T, dtype=torch.float32, device=x.device) if save_hidden else None for _ in Ns]
    n = len(Ns)
    ws_n = lib().mc_lora_group_fwd_workspace_size(ctypes.byref(d), table, n)
    ws = _workspace(ws_n, x.device)
    check(lib().mc_lora_group_fwd(ctypes.byref(d), _ptr(x), table, n, _ptr_array(ys), _ptr_array(hs), _ptr(ws), ws_n,
                                  _stream(x)))
    return ys, hs


def lora_group_backward(x, projs, dYs, scale, dropout_p=0.0, h_saves=None, need_dx=True, need_dA=True, need_dB=True):
    """Backward of lora_group_forward (mc_lora_group_bwd): returns (dX, [dA_g],
    [dB_g]) where dX [..., K] is the sum of every projection's input gradient.
    x may be None when dA is not requested (as in lora_backward); the leading
    dims then come from dYs[0] and K from the projections' A."""
    if not isinstance(dYs, (list, tuple)) or len(dYs) < 1:
        raise McError(_lib.MC_ERR_SHAPE, "one dY per projection")
    if x is None:
        if need_dA:
            raise McError(_lib.MC_ERR_NULL, "LoRA backward: dA requires x")
        if not isinstance(dYs[0], torch.Tensor) or dYs[0].dim() < 1:
            raise McError(_lib.MC_ERR_SHAPE, "dY must have at least 1 dimension")
        lead = tuple(dYs[0].shape[:-1])
        table, K, r, T, Ns = _group_table(None, projs, dropout_p, lead=lead, like=dYs[0])
    else:
        table, K, r, T, Ns = _group_table(x, projs, dropout_p)
        lead = tuple(x.shape[:-1])
    if len(dYs) != len(Ns):
        raise McError(_lib.MC_ERR_SHAPE, "one dY per projection")
    dev = dYs[0].device if x is None else x.device
    for g, (dy, N) in enumerate(zip(dYs, Ns)):
        _expect(dy, f"dY[{g}]", shape=lead + (N,), dtype=torch.bfloat16, device=dev)
    if h_saves is not None:
        for g, h in enumerate(h_saves):
            _expect(h, f"h_save[{g}]", shape=(r, T), dtype=torch.float32, device=dev)
    d = LoraDesc(T, K, Ns[0], r, float(scale), float(dropout_p), _lib.MC_BF16)
    dX = torch.empty(*lead, K, dtype=torch.bfloat16, device=dev) if need_dx else None
    dAs = [torch.empty(K, r, dtype=torch.float32, device=dev) if need_dA else None for _ in Ns]
    dBs = [torch.empty(r, N, dtype=torch.float32, device=dev) if need_dB else None for N in Ns]
    n = len(Ns)
    ws_n = lib().mc_lora_group_bwd_workspace_size(ctypes.byref(d), table, n)
    ws = _workspace(ws_n, dev)
    hp = _ptr_array(h_saves) if h_saves is not None else None
    check(lib().mc_lora_group_bwd(ctypes.byref(d), _ptr(x), table, n, hp, _ptr_array(dYs), _ptr(dX), _ptr_array(dAs),
                                  _ptr_array(dBs), _ptr(ws), ws_n, _stream(dYs[0])))
    return dX, dAs, dBs


def transpose_weight(W):
    """W^T [K, N] of a frozen bf16 base weight W [N, K] (mc_transpose_bf16):
    built once and passed as a projection's Wt, the grouped backward reads it
    instead of transposing W on every call."""
    _contig(W, "W")
    if W.dim() != 2:
        raise McError(_lib.MC_ERR_SHAPE, "W must be 2-D")
    if W.dtype != torch.bfloat16:
        raise McError(_lib.MC_ERR_DTYPE, "transpose_weight takes a bfloat16 W")
    Wt = torch.empty(W.shape[1], W.shape[0], dtype=W.dtype, device=W.device)
    check(lib().mc_transpose_bf16(W.shape[0], W.shape[1], _ptr(W), _ptr(Wt), _stream(W)))
    return Wt


def rms_norm_forward(x, eps, w=None, save_rstd=True):
    """RMSNorm over the last dim: (y, rstd). w [dim] in x's dtype or None."""
    rows, D = _rows_of(x, "x")
    _expect(w, "w", shape=(D,), dtype=x.dtype, device=x.device)
    y = torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if save_rstd else None
    check(lib().mc_rmsnorm_fwd(rows, D, float(eps), _dtype_code(x), _ptr(x), _ptr(w), _ptr(y), _ptr(rstd),
                               _stream(x)))
    return y, rstd


def rms_norm_backward(x, dy, eps, w=None, rstd=None, need_dw=True):
    """(dx, dw) of RMSNorm; rstd [rows] float32 from the forward or None."""
    rows, D = _rows_of(x, "x")
    _expect(dy, "dy", shape=x.shape, dtype=x.dtype, device=x.device)
    _expect(w, "w", shape=(D,), dtype=x.dtype, device=x.device)
    _expect(rstd, "rstd", shape=(rows,), dtype=torch.float32, device=x.device)
    dx = torch.empty_like(x)
    dw = torch.empty(D, dtype=torch.float32, device=x.device) if need_dw else None
    ws_n = lib().mc_rmsnorm_bwd_workspace_size(rows, D) if need_dw else 0
    ws = _workspace(ws_n, x.device)
    check(lib().mc_rmsnorm_bwd(rows, D, float(eps), _dtype_code(x), _ptr(x), _ptr(w), _ptr(rstd), _ptr(dy),
                               _ptr(dx), _ptr(dw), _ptr(ws), ws_n, _stream(x)))
    return dx, dw


def softmax_forward(s, causal_rows=0):
    rows, D = _rows_of(s, "s")
    p = torch.empty_like(s)
    check(lib().mc_softmax_fwd(rows, D, int(causal_rows), _dtype_code(s), _ptr(s), _ptr(p), _stream(s)))
    return p


def softmax_backward(p, dp, causal_rows=0):
    rows, D = _rows_of(p, "p")
    _expect(dp, "dp", shape=p.shape, dtype=p.dtype, device=p.device)
    ds = torch.empty_like(p)
    check(lib().mc_softmax_bwd(rows, D, int(causal_rows), _dtype_code(p), _ptr(p), _ptr(dp), _ptr(ds),
                               _stream(p)))
    return ds


def attention_desc(q, k, causal, scale):
    B, H, S, D = q.shape
    return AttnDesc(B, S, H, k.shape[1], D, int(bool(causal)), float(scale), _dtype_code(q))


def _attn_inputs(q, k, v, mask):
    """q [B, H, S, D]; k, v [B, Hkv, S, D] in q's dtype; mask fp32 [S, S] or None."""
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise McError(_lib.MC_ERR_SHAPE, "q must be [batch, heads, seq, head_dim]")
    _contig(q, "q")
    _dtype_code(q)
    B, H, S, D = q.shape
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise McError(_lib.MC_ERR_SHAPE, "k must be [batch, kv_heads, seq, head_dim]")
    Hkv = k.shape[1]
    _expect(k, "k", shape=(B, Hkv, S, D), dtype=q.dtype, device=q.device)
    _expect(v, "v", shape=(B, Hkv, S, D), dtype=q.dtype, device=q.device)
    _expect(mask, "mask", shape=(S, S), dtype=torch.float32, device=q.device)
    return B, H, S, D


def attention_forward(q, k, v, causal=False, scale=None, mask=None, save_lse=True):
    """Attention core of Attention::forward (src/models/transformer.rs:258-283):
    q [B, H, S, D], k, v [B, Hkv, S, D] -> (o [B, S, H*D], lse [B, H, S])."""
    B, H, S, D = _attn_inputs(q, k, v, mask)
    if scale is None:
        scale = D ** -0.5
    d = attention_desc(q, k, causal, scale)
    o = torch.empty(B, S, H * D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, S, dtype=torch.float32, device=q.device) if save_lse else None
    ws_n = lib().mc_attention_fwd_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, q.device)
    check(lib().mc_attention_fwd(ctypes.byref(d), _ptr(q), _ptr(k), _ptr(v), _ptr(mask), _ptr(o), _ptr(lse),
                                 _ptr(ws), ws_n, _stream(q)))
    return o, lse


def attention_backward(q, k, v, o, lse, dout, causal=False, scale=None, mask=None):
    """(dq, dk, dv) of attention_forward; o and lse come from the forward."""
    B, H, S, D = _attn_inputs(q, k, v, mask)
    _expect(o, "o", shape=(B, S, H * D), dtype=q.dtype, device=q.device)
    _expect(dout, "dout", shape=(B, S, H * D), dtype=q.dtype, device=q.device)
    _expect(lse, "lse", shape=(B, H, S), dtype=torch.float32, device=q.device)
    if o is None or lse is None or dout is None:
        raise McError(_lib.MC_ERR_NULL, "attention backward: o, lse and dout are required")
    if scale is None:
        scale = D ** -0.5
    d = attention_desc(q, k, causal, scale)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws_n = lib().mc_attention_bwd_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, q.device)
    check(lib().mc_attention_bwd(ctypes.byref(d), _ptr(q), _ptr(k), _ptr(v), _ptr(mask), _ptr(o), _ptr(lse),
                                 _ptr(dout), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), ws_n, _stream(q)))
    return dq, dk, dv


def attention_spans(documents=None, prefix=None, causal=True):
    """Who sees whom in rows that hold several documents: int32 [B, S, 4], made once for every layer's
    packed_attention_forward and _backward.

    documents int32 [B, S]: a document is a run of equal ids, whose tokens see each other only; ids below 0 are
    padding, which sees nothing and is not seen (None: a row is one document). causal: a token sees those up to
    itself; prefix uint8 or bool [B, S] then marks prompts, a document's leading tokens, which also see each other
    (non-zero tokens behind a document's first zero are no prompt). A token's entry holds the keys that it sees as a
    query, from and to, then the queries that see it as a key."""
    ref = documents if documents is not None else prefix
    if ref is None:
        raise McError(_lib.MC_ERR_NULL, "attention_spans: documents or prefix is required (without either, call the "
                      "attention with causal)")
    if not isinstance(ref, torch.Tensor) or ref.dim() != 2 or ref.numel() == 0:
        raise McError(_lib.MC_ERR_SHAPE, "documents and prefix must be [batch, seq]")
    dev, shape = ref.device, tuple(ref.shape)
    ids = _address(documents, "documents", shape, torch.int32, dev)
    if isinstance(prefix, torch.Tensor) and prefix.dtype == torch.bool:
        prefix = prefix.view(torch.uint8)
    flags = _address(prefix, "prefix", shape, torch.uint8, dev)
    spans = torch.empty(*shape, 4, dtype=torch.int32, device=dev)
    _launch(ref, lib().mc_attention_spans, *shape, ids, flags, int(bool(causal)), spans.data_ptr())
    return spans


def _packed_call(q, k, v, spans, causal, scale, cap, slopes):
    B, H, S, D = _attn_inputs(q, k, v, None)
    if spans is not None and causal:
        raise McError(_lib.MC_ERR_VALUE, "causal must be False with spans, which hold it")
    at = _address(spans, "spans", (B, S, 4), torch.int32, q.device)
    by = _address(slopes, "slopes", (H,), torch.float32, q.device)
    d = PackedAttnDesc(attention_desc(q, k, causal, D ** -0.5 if scale is None else scale),
                       0.0 if cap is None else float(cap), 0)
    return d, at, by


def packed_attention_forward(q, k, v, spans=None, causal=False, scale=None, cap=None, slopes=None, save_lse=True):
    """Attention over packed rows, with capped scores and a bias by distance: (o [B, S, H*D], lse [B, H, S]).

    q [B, H, S, D], k and v [B, Hkv, S, D]. spans from attention_spans say who sees whom; without them causal does.
    The scores are x = scale q.k, then cap * tanh(x / cap) (cap in [0.01, 1000]; None: uncapped), then
    x - slopes[h] * |i - j| (slopes fp32 [H], constants; None: none). A query that sees nothing has o = 0 and
    lse = -inf. What is hidden may hold anything, NaN included. scale > 0, default 1 / sqrt(D)."""
    d, at, by = _packed_call(q, k, v, spans, causal, scale, cap, slopes)
    B, H, S, D = q.shape
    o = torch.empty(B, S, H * D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, S, dtype=torch.float32, device=q.device) if save_lse else None
    ws_n = lib().mc_packed_attention_fwd_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, q.device)
    _launch(q, lib().mc_packed_attention_fwd, ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), at, by,
            o.data_ptr(), _ptr(lse), _ptr(ws), ws_n)
    return o, lse


def packed_attention_backward(q, k, v, o, lse, dout, spans=None, causal=False, scale=None, cap=None, slopes=None):
    """(dq, dk, dv) of packed_attention_forward, called as it was; o and lse come from it. Padding gets zeros."""
    d, at, by = _packed_call(q, k, v, spans, causal, scale, cap, slopes)
    B, H, S, D = q.shape
    if o is None or lse is None or dout is None:
        raise McError(_lib.MC_ERR_NULL, "packed attention backward: o, lse and dout are required")
    o_at = _address(o, "o", (B, S, H * D), q.dtype, q.device)
    g_at = _address(dout, "dout", (B, S, H * D), q.dtype, q.device)
    lse_at = _address(lse, "lse", (B, H, S), torch.float32, q.device)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws_n = lib().mc_packed_attention_bwd_workspace_size(ctypes.byref(d), int(at is not None))
    ws = _workspace(ws_n, q.device)
    _launch(q, lib().mc_packed_attention_bwd, ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), at, by, o_at,
            lse_at, g_at, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), ws_n)
    return dq, dk, dv


def layer_norm_forward(x, eps, w=None, b=None, save_stats=True):
    """LayerNorm over the last dim: (y, mean, rstd). w, b [dim] in x's dtype or None."""
    rows, D = _rows_of(x, "x")
    _expect(w, "w", shape=(D,), dtype=x.dtype, device=x.device)
    _expect(b, "b", shape=(D,), dtype=x.dtype, device=x.device)
    y = torch.empty_like(x)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device) if save_stats else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if save_stats else None
    check(lib().mc_layernorm_fwd(rows, D, float(eps), _dtype_code(x), _ptr(x), _ptr(w), _ptr(b), _ptr(y), _ptr(mean),
                                 _ptr(rstd), _stream(x)))
    return y, mean, rstd


def layer_norm_backward(x, dy, eps, w=None, mean=None, rstd=None, need_dw=True, need_db=True):
    """(dx, dw, db) of LayerNorm; dw / db are fp32 [D] (None when not requested)."""
    rows, D = _rows_of(x, "x")
    _expect(dy, "dy", shape=x.shape, dtype=x.dtype, device=x.device)
    _expect(w, "w", shape=(D,), dtype=x.dtype, device=x.device)
    _expect(mean, "mean", shape=(rows,), dtype=torch.float32, device=x.device)
    _expect(rstd, "rstd", shape=(rows,), dtype=torch.float32, device=x.device)
    dx = torch.empty_like(x)
    dw = torch.empty(D, dtype=torch.float32, device=x.device) if need_dw else None
    db = torch.empty(D, dtype=torch.float32, device=x.device) if need_db else None
    ws_n = lib().mc_layernorm_bwd_workspace_size(rows, D) if (need_dw or need_db) else 0
    ws = _workspace(ws_n, x.device)
    check(lib().mc_layernorm_bwd(rows, D, float(eps), _dtype_code(x), _ptr(x), _ptr(w), _ptr(mean), _ptr(rstd),
                                 _ptr(dy), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), ws_n, _stream(x)))
    return dx, dw, db


def log_softmax_forward(x):
    rows, D = _rows_of(x, "x")
    y = torch.empty_like(x)
    check(lib().mc_log_softmax_fwd(rows, D, _dtype_code(x), _ptr(x), _ptr(y), _stream(x)))
    return y


def log_softmax_backward(y, dy):
    rows, D = _rows_of(y, "y")
    _expect(dy, "dy", shape=y.shape, dtype=y.dtype, device=y.device)
    dx = torch.empty_like(y)
    check(lib().mc_log_softmax_bwd(rows, D, _dtype_code(y), _ptr(y), _ptr(dy), _ptr(dx), _stream(y)))
    return dx


def _xent_desc(logits, ignore_index, smoothing):
    rows, V = _rows_of(logits, "logits")
    return XentDesc(rows, V, -1 if ignore_index is None else int(ignore_index), float(smoothing),
                    _dtype_code(logits))


def _targets(targets, logits):
    """uint32 targets [rows] as the kernels read them: torch.uint32, or
    torch.int32 (the same bytes for ids below 2^31); int64 ids are converted
    explicitly (a copy), so their low 32 bits are what the kernels see."""
    rows = logits.numel() // logits.shape[-1]
    if not isinstance(targets, torch.Tensor):
        raise McError(_lib.MC_ERR_NULL, "targets must be a tensor")
    if targets.dtype == torch.int64:
        targets = targets.to(torch.int32)
    if targets.dtype not in (torch.int32, torch.uint32):
        raise McError(_lib.MC_ERR_DTYPE, f"targets have dtype {targets.dtype}, expected uint32 (or int32 / int64 ids)")
    _expect(targets, "targets", device=logits.device)
    if targets.numel() != rows:
        raise McError(_lib.MC_ERR_SHAPE, f"targets have {targets.numel()} entries, expected {rows} (one per row)")
    return targets


def cross_entropy_forward(logits, targets, ignore_index=None, smoothing=0.0):
    """cross_entropy_loss (src/training/loss.rs:58-245) over logits [..., V] and
    uint32 targets [...]: (loss fp32 [1], stats fp32 [rows + 1])."""
    d = _xent_desc(logits, ignore_index, smoothing)
    targets = _targets(targets, logits)
    loss = torch.empty(1, dtype=torch.float32, device=logits.device)
    stats = torch.empty(d.rows + 1, dtype=torch.float32, device=logits.device)
    ws_n = lib().mc_cross_entropy_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, logits.device)
    check(lib().mc_cross_entropy_fwd(ctypes.byref(d), _ptr(logits), _ptr(targets), _ptr(loss), _ptr(stats), _ptr(ws),
                                     ws_n, _stream(logits)))
    return loss, stats


def cross_entropy_backward(logits, targets, stats, dloss=None, ignore_index=None, smoothing=0.0):
    """d loss / d logits (times dloss, a fp32 [1] device tensor; default 1)."""
    d = _xent_desc(logits, ignore_index, smoothing)
    targets = _targets(targets, logits)
    _expect(stats, "stats", shape=(d.rows + 1,), dtype=torch.float32, device=logits.device)
    if stats is None:
        raise McError(_lib.MC_ERR_NULL, "stats from cross_entropy_forward are required")
    if dloss is None:
        dloss = torch.ones(1, dtype=torch.float32, device=logits.device)
    _expect(dloss, "dloss", shape=(1,), dtype=torch.float32, device=logits.device)
    dlogits = torch.empty_like(logits)
    check(lib().mc_cross_entropy_bwd(ctypes.byref(d), _ptr(logits), _ptr(targets), _ptr(stats), _ptr(dloss),
                                     _ptr(dlogits), _stream(logits)))
    return dlogits


# --------------------------------------------------- losses over log-probabilities
def _address(t, name, shape, dtype, device):
    """The device address of a tensor of the given shape (a tuple), or None for None."""
    if t is None:
        return None
    if type(t) is not torch.Tensor or t.shape != shape or t.dtype is not dtype or t.device != device or \
            not t.is_contiguous():
        _expect(t, name, shape, dtype, device)
    return t.data_ptr()


def _launch(t, fn, *args):
    """fn(*args, stream) on the device of t and its current stream."""
    if not t.is_cuda:
        torch.cuda.current_stream(t.device)  # refuses what is not on a GPU
    device = t.get_device()
    if device != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    check(status)


def _loss_inputs(logits, targets, ignore_index, seqs):
    """(targets as the kernels read them, ignore_index, dtype code) of logits [..., V] with targets over its leading
    dims; seqs: the logits must be [sequences, tokens, V]. Targets are unsigned: an ignore_index below 0 is none, as
    for the cross entropy, and padding of -100 is 2**32 - 100 there."""
    if not isinstance(logits, torch.Tensor):
        raise McError(_lib.MC_ERR_NULL, "logits must be a tensor")
    if seqs and logits.dim() != 3:
        raise McError(_lib.MC_ERR_SHAPE, f"logits must be [sequences, tokens, vocab], got {tuple(logits.shape)}")
    _rows_of(logits, "logits")
    if logits.numel() == 0:
        raise McError(_lib.MC_ERR_SHAPE, f"logits are empty: {tuple(logits.shape)}")
    targets = _targets(targets, logits)
    if seqs and targets.shape != logits.shape[:-1]:
        raise McError(_lib.MC_ERR_SHAPE,
                      f"targets has shape {tuple(targets.shape)}, expected {tuple(logits.shape[:-1])}")
    return targets, -1 if ignore_index is None else int(ignore_index), _DTYPES[logits.dtype]


def _logprob_desc(logits, ignore, temperature, code):
    V = logits.shape[-1]
    return LogprobDesc(logits.numel() // V, V, ignore, float(temperature), code)


def token_logprobs_forward(logits, targets, ignore_index=None, temperature=1.0, save_stats=True):
    """Log-probabilities of the given tokens under logits [..., V]: (logps [...] fp32, stats). targets hold one id per
    row of logits, in any shape.

    logps = logits[target] / T - logsumexp(logits / T), 0 where the target is
    ignore_index (such rows are not read); stats [rows, 2] fp32 is what
    token_logprobs_backward needs, or None. Here and in the other losses
    targets are read as 32-bit unsigned ids and an ignore_index below 0 is
    none: padding of -100 takes ignore_index=2**32 - 100, or its rows are NaN."""
    targets, ignore, code = _loss_inputs(logits, targets, ignore_index, False)
    d = _logprob_desc(logits, ignore, temperature, code)
    if targets.shape == logits.shape[:-1]:
        logps = torch.empty_like(targets, dtype=torch.float32)  # half the time of empty with a shape
    else:
        logps = torch.empty(logits.shape[:-1], dtype=torch.float32, device=logits.device)
    stats = torch.empty(d.rows, 2, dtype=torch.float32, device=logits.device) if save_stats else None
    ws_n = lib().mc_token_logprobs_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, logits.device)
    _launch(logits, lib().mc_token_logprobs_fwd, ctypes.byref(d), logits.data_ptr(), targets.data_ptr(),
            logps.data_ptr(), _ptr(stats), _ptr(ws), ws_n)
    return logps, stats


def token_logprobs_backward(logits, targets, stats, dlogps, ignore_index=None, temperature=1.0):
    """The logits' gradient from that of their tokens' log-probabilities, dlogps [...] fp32: with it, any loss over
    log-probabilities has its gradient in one pass over the logits."""
    targets, ignore, code = _loss_inputs(logits, targets, ignore_index, False)
    d = _logprob_desc(logits, ignore, temperature, code)
    dev = logits.device
    if stats is None or dlogps is None:
        raise McError(_lib.MC_ERR_NULL, "token_logprobs_backward: stats and dlogps are required")
    stats_at = _address(stats, "stats", (d.rows, 2), torch.float32, dev)
    dlogps_at = _address(dlogps, "dlogps", logits.shape[:-1], torch.float32, dev)
    dlogits = torch.empty_like(logits)
    _launch(logits, lib().mc_token_logprobs_bwd, ctypes.byref(d), logits.data_ptr(), targets.data_ptr(), stats_at,
            dlogps_at, dlogits.data_ptr())
    return dlogits


_PREF_KINDS = {"sigmoid": _lib.MC_PREF_SIGMOID, "hinge": _lib.MC_PREF_HINGE, "squared": _lib.MC_PREF_SQUARED}


def _choice(table, key, name):
    try:
        return table[key]
    except (KeyError, TypeError):
        raise McError(_lib.MC_ERR_VALUE, f"{name} must be one of {', '.join(table)}, got {key!r}")


def _pairs(logits):
    if logits.shape[0] % 2:
        raise McError(_lib.MC_ERR_SHAPE, f"logits hold pairs of sequences: {logits.shape[0]} is odd")
    return logits.shape[0] // 2


def preference_loss_forward(logits, targets, ref_logps=None, beta=0.1, kind="sigmoid", label_smoothing=0.0, margin=0.0,
                            average=False, ignore_index=None):
    """Preference loss over pairs of sequences: (loss [1], rewards [2P], stats).

    logits [2P, S, V], the P preferred answers first, then the others in the
    same order; targets [2P, S], padding and prompts as ignore_index; ref_logps
    [2P, S] fp32, the reference policy's token_logprobs_forward (None: no
    reference). A sequence's score is the sum (average: the mean) of logps -
    ref_logps, d a pair's difference of scores, z = beta d - margin; the loss
    is the pairs' mean of -(1 - e) log sigma(z) - e log sigma(-z) with
    e = label_smoothing ("sigmoid"), max(0, 1 - z) ("hinge") or
    (d - 1 / (2 beta))^2 ("squared"). rewards = beta times the scores."""
    targets, ignore, code = _loss_inputs(logits, targets, ignore_index, True)
    P, dev = _pairs(logits), logits.device
    _, S, V = logits.shape
    d = PreferenceDesc(P, S, V, ignore, _choice(_PREF_KINDS, kind, "kind"), int(bool(average)), float(beta),
                       float(label_smoothing), float(margin), code)
    ref = _address(ref_logps, "ref_logps", (2 * P, S), torch.float32, dev)
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    rewards = torch.empty(2 * P, dtype=torch.float32, device=dev)
    stats = torch.empty(4 * P * S + 2 * P, dtype=torch.float32, device=dev)
    ws_n = lib().mc_preference_loss_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, dev)
    _launch(logits, lib().mc_preference_loss_fwd, ctypes.byref(d), logits.data_ptr(), targets.data_ptr(), ref,
            loss.data_ptr(), rewards.data_ptr(), stats.data_ptr(), _ptr(ws), ws_n)
    return loss, rewards, stats


def preference_loss_backward(logits, targets, stats, dloss=None, ignore_index=None):
    """d loss / d logits (times dloss, a fp32 [1] device tensor; default 1); stats from preference_loss_forward."""
    targets, ignore, code = _loss_inputs(logits, targets, ignore_index, True)
    P, dev = _pairs(logits), logits.device
    _, S, V = logits.shape
    if stats is None:
        raise McError(_lib.MC_ERR_NULL, "stats from preference_loss_forward are required")
    _expect(stats, "stats", (4 * P * S + 2 * P,), torch.float32, dev)
    g = _address(dloss, "dloss", (1,), torch.float32, dev)
    # what the loss was is in stats
    d = PreferenceDesc(P, S, V, ignore, _lib.MC_PREF_SIGMOID, 0, 1.0, 0.0, 0.0, code)
    dlogits = torch.empty_like(logits)
    _launch(logits, lib().mc_preference_loss_bwd, ctypes.byref(d), logits.data_ptr(), targets.data_ptr(),
            stats.data_ptr(), g, dlogits.data_ptr())
    return dlogits


_REDUCTIONS = {"tokens": _lib.MC_MEAN_TOKENS, "sequences": _lib.MC_MEAN_SEQUENCES}


def _policy_call(logits, targets, advantages, old_logps, ref_logps, clip_low, clip_high, kl_coef, temperature,
                 reduction, ignore_index):
    targets, ignore, code = _loss_inputs(logits, targets, ignore_index, True)
    B, S, V = logits.shape
    dev = logits.device
    if not isinstance(advantages, torch.Tensor):
        raise McError(_lib.MC_ERR_NULL, "advantages must be a tensor")
    per_token = advantages.dim() == 2
    _address(advantages, "advantages", (B, S) if per_token else (B,), torch.float32, dev)
    old = _address(old_logps, "old_logps", (B, S), torch.float32, dev)
    ref = _address(ref_logps, "ref_logps", (B, S), torch.float32, dev)
    d = PolicyDesc(B, S, V, ignore, int(per_token), _choice(_REDUCTIONS, reduction, "reduction"), float(clip_low),
                   float(clip_high), float(kl_coef), float(temperature), code)
    loss, metrics = (torch.empty(n, dtype=torch.float32, device=dev) for n in (1, 2))
    return d, targets, old, ref, loss, torch.empty_like(targets, dtype=torch.float32), metrics


def policy_loss_forward(logits, targets, advantages, old_logps=None, ref_logps=None, clip_low=0.2, clip_high=0.2,
                        kl_coef=0.0, temperature=1.0, reduction="tokens", ignore_index=None):
    """Clipped policy loss over sampled tokens: (loss [1], logps [B, S], metrics [2], stats).

    logits [B, S, V], targets [B, S] (padding and prompts as ignore_index),
    advantages [B] or [B, S] fp32; old_logps and ref_logps [B, S] fp32, the
    sampling and the reference policy's token_logprobs_forward at the same
    temperature. With r = exp(logps - old_logps) (1 without old_logps) a token's
    loss is -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef kl,
    kl = exp(ref - logps) - (ref - logps) - 1; the loss is their mean over the
    counted tokens, or with reduction="sequences" the batch's mean of the
    sequences' means. metrics: kl and the share of clipped tokens, averaged
    alike."""
    d, targets, old, ref, loss, logps, metrics = _policy_call(
        logits, targets, advantages, old_logps, ref_logps, clip_low, clip_high, kl_coef, temperature, reduction,
        ignore_index)
    stats = torch.empty(3 * logps.numel() + 1, dtype=torch.float32, device=logits.device)
    ws_n = lib().mc_policy_loss_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, logits.device)
    _launch(logits, lib().mc_policy_loss_fwd, ctypes.byref(d), logits.data_ptr(), targets.data_ptr(),
            advantages.data_ptr(), old, ref, loss.data_ptr(), logps.data_ptr(), metrics.data_ptr(), stats.data_ptr(),
            _ptr(ws), ws_n)
    return loss, logps, metrics, stats


def policy_loss_backward(logits, targets, stats, dloss=None, temperature=1.0, ignore_index=None):
    """d loss / d logits (times dloss, a fp32 [1] device tensor; default 1); stats from policy_loss_forward."""
    targets, ignore, code = _loss_inputs(logits, targets, ignore_index, True)
    B, S, V = logits.shape
    dev = logits.device
    if stats is None:
        raise McError(_lib.MC_ERR_NULL, "stats from policy_loss_forward are required")
    _expect(stats, "stats", (3 * B * S + 1,), torch.float32, dev)
    g = _address(dloss, "dloss", (1,), torch.float32, dev)
    d = PolicyDesc(B, S, V, ignore, 0, _lib.MC_MEAN_TOKENS, 0.0, 0.0, 0.0, float(temperature), code)
    dlogits = torch.empty_like(logits)
    _launch(logits, lib().mc_policy_loss_bwd, ctypes.byref(d), logits.data_ptr(), targets.data_ptr(), stats.data_ptr(),
            g, dlogits.data_ptr())
    return dlogits


def policy_loss_forward_backward(logits, targets, advantages, old_logps=None, ref_logps=None, clip_low=0.2,
                                 clip_high=0.2, kl_coef=0.0, temperature=1.0, reduction="tokens", ignore_index=None,
                                 dloss=None):
    """policy_loss_forward and _backward in one call, for a training step: (loss, logps, metrics, dlogits). The
    logits need not be read twice."""
    d, targets, old, ref, loss, logps, metrics = _policy_call(
        logits, targets, advantages, old_logps, ref_logps, clip_low, clip_high, kl_coef, temperature, reduction,
        ignore_index)
    g = _address(dloss, "dloss", (1,), torch.float32, logits.device)
    dlogits = torch.empty_like(logits)
    ws_n = lib().mc_policy_loss_fwd_bwd_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, logits.device)
    _launch(logits, lib().mc_policy_loss_fwd_bwd, ctypes.byref(d), logits.data_ptr(), targets.data_ptr(),
            advantages.data_ptr(), old, ref, g, loss.data_ptr(), logps.data_ptr(), metrics.data_ptr(),
            dlogits.data_ptr(), _ptr(ws), ws_n)
    return loss, logps, metrics, dlogits


def _distill_call(logits, teacher_ids, teacher_logits, temperature, teacher_lse, mask):
    rows, V = _rows_of(logits, "logits")
    lead, dev = tuple(logits.shape[:-1]), logits.device
    if not isinstance(teacher_ids, torch.Tensor) or not isinstance(teacher_logits, torch.Tensor):
        raise McError(_lib.MC_ERR_NULL, "teacher_ids and teacher_logits must be tensors")
    if teacher_ids.dim() != logits.dim() or tuple(teacher_ids.shape[:-1]) != lead:
        raise McError(_lib.MC_ERR_SHAPE,
                      f"teacher_ids has shape {tuple(teacher_ids.shape)}, expected {lead} and the number of entries")
    K = teacher_ids.shape[-1]
    if teacher_ids.dtype == torch.int64:
        # ids that do not fit 32 bits stay out of every vocabulary
        teacher_ids = teacher_ids.clamp(-1, 2**31 - 1).to(torch.int32)
    _expect(teacher_ids, "teacher_ids", lead + (K,), torch.int32, dev)
    _expect(teacher_logits, "teacher_logits", lead + (K,), torch.float32, dev)
    lse = _address(teacher_lse, "teacher_lse", lead, torch.float32, dev)
    m = _address(mask, "mask", lead, torch.uint8, dev)
    return DistillDesc(rows, V, K, float(temperature), _DTYPES[logits.dtype]), teacher_ids, lse, m


def distillation_loss_forward(logits, teacher_ids, teacher_logits, temperature=1.0, teacher_lse=None, mask=None):
    """Distillation from a teacher's top logits: (loss [1], stats).

    logits [..., V]; teacher_ids int32 and teacher_logits fp32 [..., K], K up to
    256, in any order (an entry of -inf is left out, whatever its id); mask
    uint8 [...], rows of 0 are not counted. p = softmax(teacher_logits / T), or
    exp(teacher_logits / T - teacher_lse) where teacher_lse [...] holds the
    log-sum-exp of all the teacher's logits / T (T as a float32); the loss is T^2
    times the counted rows' mean of sum_k p_k (log p_k - log softmax(logits / T)[id_k])."""
    d, ids, lse, m = _distill_call(logits, teacher_ids, teacher_logits, temperature, teacher_lse, mask)
    dev = logits.device
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    stats = torch.empty(2 * d.rows + 1, dtype=torch.float32, device=dev)
    ws_n = lib().mc_distill_loss_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, dev)
    _launch(logits, lib().mc_distill_loss_fwd, ctypes.byref(d), logits.data_ptr(), ids.data_ptr(),
            teacher_logits.data_ptr(), lse, m, loss.data_ptr(), stats.data_ptr(), _ptr(ws), ws_n)
    return loss, stats


def distillation_loss_backward(logits, teacher_ids, teacher_logits, stats, dloss=None, temperature=1.0,
                               teacher_lse=None, mask=None):
    """d loss / d logits (times dloss, a fp32 [1] device tensor; default 1); stats from distillation_loss_forward."""
    d, ids, lse, m = _distill_call(logits, teacher_ids, teacher_logits, temperature, teacher_lse, mask)
    dev = logits.device
    if stats is None:
        raise McError(_lib.MC_ERR_NULL, "stats from distillation_loss_forward are required")
    _expect(stats, "stats", (2 * d.rows + 1,), torch.float32, dev)
    g = _address(dloss, "dloss", (1,), torch.float32, dev)
    dlogits = torch.empty_like(logits)
    _launch(logits, lib().mc_distill_loss_bwd, ctypes.byref(d), logits.data_ptr(), ids.data_ptr(),
            teacher_logits.data_ptr(), lse, m, stats.data_ptr(), g, dlogits.data_ptr())
    return dlogits


def distillation_loss_forward_backward(logits, teacher_ids, teacher_logits, temperature=1.0, teacher_lse=None,
                                       mask=None, dloss=None):
    """distillation_loss_forward and _backward in one call, for a training step: (loss, dlogits). The logits need not
    be read twice."""
    d, ids, lse, m = _distill_call(logits, teacher_ids, teacher_logits, temperature, teacher_lse, mask)
    dev = logits.device
    g = _address(dloss, "dloss", (1,), torch.float32, dev)
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    dlogits = torch.empty_like(logits)
    ws_n = lib().mc_distill_loss_fwd_bwd_workspace_size(ctypes.byref(d))
    ws = _workspace(ws_n, dev)
    _launch(logits, lib().mc_distill_loss_fwd_bwd, ctypes.byref(d), logits.data_ptr(), ids.data_ptr(),
            teacher_logits.data_ptr(), lse, m, g, loss.data_ptr(), dlogits.data_ptr(), _ptr(ws), ws_n)
    return loss, dlogits


# ------------------------------------------------------------------ embedding
def _ids(ids, device):
    """int32 ids, as the kernels read them; int64 ids are converted (a copy), those that do not fit to one that is in
    no table."""
    if not isinstance(ids, torch.Tensor):
        raise McError(_lib.MC_ERR_NULL, "ids must be a tensor")
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, 2**31 - 1).to(torch.int32)
    _expect(ids, "ids", dtype=torch.int32, device=device)
    if ids.numel() == 0:
        raise McError(_lib.MC_ERR_SHAPE, "ids are empty")
    return ids


def _padding(padding_id):
    """The id of padding, -1 for none. Ids past int32 arrive as 2**31 - 1, which is in no table and no padding."""
    if padding_id is None or padding_id < 0:
        return -1
    if padding_id > 2**31 - 2:
        raise McError(_lib.MC_ERR_VALUE, f"padding_id must be below 2**31 - 1, got {padding_id}")
    return int(padding_id)


def embedding_forward(table, ids, scale=1.0, padding_id=None):
    """scale * table[ids] for table [V, D] and ids int32 (or int64) [...]: [..., D] in the table's dtype, rounded once.

    A token of padding_id gets zeros, one whose id is not in the table NaN. padding_id None or below 0: none (a token of
    a negative id gets NaN then too)."""
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.numel() == 0:
        raise McError(_lib.MC_ERR_SHAPE, "table must be [vocab, dim]")
    _contig(table, "table")
    code = _dtype_code(table)
    ids = _ids(ids, table.device)
    V, D = table.shape
    d = EmbeddingDesc(ids.numel(), V, D, _padding(padding_id), float(scale), code)
    out = torch.empty(*ids.shape, D, dtype=table.dtype, device=table.device)
    _launch(table, lib().mc_embedding_fwd, ctypes.byref(d), table.data_ptr(), ids.data_ptr(), out.data_ptr())
    return out


def embedding_backward(dout, ids, vocab, scale=1.0, padding_id=None, dtable=None):
    """The table's gradient [vocab, D] fp32: scale times the sum of dout [..., D] over the tokens of each id.

    Without dtable a new one, zero for ids that do not occur; with it (fp32 [vocab, D]) the sums are added to it, as
    where the table is the output projection's weight as well. Padding, and ids that are not in the table, are left
    out. The sums run in a fixed order."""
    if not isinstance(dout, torch.Tensor) or dout.dim() < 2 or dout.numel() == 0:
        raise McError(_lib.MC_ERR_SHAPE, "dout must be [..., dim], one row per id")
    _contig(dout, "dout")
    code = _dtype_code(dout)
    ids = _ids(ids, dout.device)
    if ids.shape != dout.shape[:-1]:
        raise McError(_lib.MC_ERR_SHAPE, f"ids has shape {tuple(ids.shape)}, expected {tuple(dout.shape[:-1])}")
    D, V = dout.shape[-1], int(vocab)
    d = EmbeddingDesc(ids.numel(), V, D, _padding(padding_id), float(scale), code)
    into = _address(dtable, "dtable", (V, D), torch.float32, dout.device)
    ws_n = lib().mc_embedding_bwd_workspace_size(ctypes.byref(d))
    if dtable is None and ws_n:
        dtable = torch.empty(V, D, dtype=torch.float32, device=dout.device)
    ws = _workspace(ws_n, dout.device)
    _launch(dout, lib().mc_embedding_bwd, ctypes.byref(d), ids.data_ptr(), dout.data_ptr(), _ptr(dtable),
            int(into is not None), _ptr(ws), ws_n)
    return dtable


# ------------------------------------------------------- gradients' norm, AdamW
def _tensors(group, name):
    """(dtypes, sizes, addresses, device) of a list of contiguous tensors of one device. One pass over the list per
    property: a model's adapters are hundreds of small tensors, and their checks take longer than their kernels."""
    if not isinstance(group, (list, tuple)) or not group:
        raise McError(_lib.MC_ERR_SHAPE, f"{name} must be a list of at least one tensor")
    try:
        whole = all(map(torch.Tensor.is_contiguous, group))
    except TypeError:
        raise McError(_lib.MC_ERR_NULL, f"{name} must hold tensors only")
    if not whole:
        raise McError(_lib.MC_ERR_LAYOUT, f"every tensor of {name} must be contiguous")
    dtypes = list(map(_DTYPE_OF, group))
    for dtype in set(dtypes):
        if dtype not in _DTYPES:
            raise McError(_lib.MC_ERR_DTYPE, f"unsupported dtype {dtype} in {name} (float32 or bfloat16)")
    indices = set(map(torch.Tensor.get_device, group))
    if len(indices) > 1 or -1 in indices:  # the device objects take twice the time
        devices = {t.device for t in group}
        if len(devices) > 1:
            raise McError(_lib.MC_ERR_LAYOUT, f"{name} are on {len(devices)} devices, expected one")
    return dtypes, list(map(torch.Tensor.numel, group)), list(map(torch.Tensor.data_ptr, group)), group[0].device


def _grad_table(grads, outs, written=True):
    """(address of the mc_grad_tensor table, its length, what keeps it alive) of gradients and where they go."""
    dtypes, sizes, at, device = _tensors(grads, "grads")
    to, out_dtypes = at, dtypes
    if outs is not None and outs is not grads:
        if len(outs) != len(grads):
            raise McError(_lib.MC_ERR_SHAPE, f"outs list has {len(outs)} entries, expected {len(grads)}")
        out_dtypes, out_sizes, to, out_device = _tensors(outs, "outs")
        if out_sizes != sizes:
            i = next(i for i, (a, b) in enumerate(zip(sizes, out_sizes)) if a != b)
            raise McError(_lib.MC_ERR_SHAPE, f"outs[{i}] has {out_sizes[i]} elements, expected {sizes[i]}")
        if out_device != device:
            raise McError(_lib.MC_ERR_LAYOUT, f"outs are on {out_device}, expected {device}")
    if written and len(set(to)) < len(to) and len({p for p, n in zip(to, sizes) if n}) < sum(map(bool, sizes)):
        raise McError(_lib.MC_ERR_LAYOUT, "a tensor is listed twice: it would be scaled twice")
    if len(set(dtypes)) == 1 and len(set(out_dtypes)) == 1:
        codes = itertools.repeat(_DTYPES[dtypes[0]] | _DTYPES[out_dtypes[0]] << 32)
    else:
        codes = [_DTYPES[a] | _DTYPES[b] << 32 for a, b in zip(dtypes, out_dtypes)]
    table = array.array("Q", itertools.chain.from_iterable(zip(at, to, sizes, codes)))
    return table.buffer_info()[0], len(sizes), table


def gradient_norm(grads, max_norm=None):
    """The global norm of a list of fp32 or bf16 gradients, and the factor that brings it to max_norm: (norm [1],
    scale [1]), fp32 on the device; scale is None without max_norm.

    norm = sqrt(sum of all squares), summed in 64 bits in a fixed order; scale = 1 where norm <= max_norm, else
    max_norm / norm. Pass scale to scale_gradients, or to adamw_step, which then clips as it reads."""
    at, n, table = _grad_table(grads, None, written=False)
    dev = grads[0].device
    norm = torch.empty(1, dtype=torch.float32, device=dev)
    scale = None if max_norm is None else torch.empty(1, dtype=torch.float32, device=dev)
    ws_n = lib().mc_gradient_norm_workspace_size(at, n)
    ws = _workspace(ws_n, dev)
    _launch(grads[0], lib().mc_gradient_norm, at, n, 1.0 if max_norm is None else float(max_norm), norm.data_ptr(),
            _ptr(scale), _ptr(ws), ws_n)
    return norm, scale


def scale_gradients(grads, scale, outs=None):
    """Every gradient times scale (fp32 [1] on the device) into outs (fp32 or bf16 tensors of the same sizes; default:
    in place), one rounding each. An output is its own gradient or apart from every gradient and output: one that is
    listed twice, or overlaps another, is refused. Returns outs."""
    at, n, table = _grad_table(grads, outs)
    if scale is None:
        raise McError(_lib.MC_ERR_NULL, "scale must be a tensor")
    _expect(scale, "scale", (1,), torch.float32, grads[0].device)
    _launch(grads[0], lib().mc_scale_gradients, at, n, scale.data_ptr())
    return grads if outs is None else outs


def clip_gradients(grads, max_norm, outs=None):
    """gradient_norm and scale_gradients in one call: (norm [1], scale [1]). outs may have another dtype than the
    gradients, as fp32 ones for adamw_step from bf16 ones."""
    at, n, table = _grad_table(grads, outs)
    dev = grads[0].device
    norm, scale = (torch.empty(1, dtype=torch.float32, device=dev) for _ in range(2))
    ws_n = lib().mc_gradient_norm_workspace_size(at, n)
    ws = _workspace(ws_n, dev)
    _launch(grads[0], lib().mc_clip_gradients, at, n, float(max_norm), norm.data_ptr(), scale.data_ptr(), _ptr(ws), ws_n)
    return norm, scale


def adamw_step(params, grads, ms, vs, steps, lr=1e-4, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
               outs=None, grad_scale=None):
    """AdamW::step (src/training/optimizer.rs:227-281) for a list of fp32
    tensors in one call: m and v are updated in place; the new parameters go
    to outs (default: the params themselves, in place). steps: one step count
    per tensor (or one int for all). grad_scale: gradient_norm's scale (fp32 [1]
    on the device), by which every gradient is multiplied first, as
    scale_gradients would, without writing it."""
    n = len(params)
    if isinstance(steps, int):
        steps = [steps] * n
    outs = params if outs is None else outs
    for group, name in ((params, "param"), (grads, "grad"), (ms, "m"), (vs, "v"), (outs, "param_out")):
        if len(group) != n:
            raise McError(_lib.MC_ERR_SHAPE, f"{name} list has {len(group)} entries, expected {n}")
        for t in group:
            _contig(t, name)
            if t.dtype != torch.float32:
                raise McError(_lib.MC_ERR_DTYPE, f"{name} must be float32")
    table = (AdamWTensor * max(n, 1))()
    for i in range(n):
        numel = params[i].numel()
        for t in (grads[i], ms[i], vs[i], outs[i]):
            if t.numel() != numel:
                raise McError(_lib.MC_ERR_SHAPE, f"tensor {i}: element counts differ")
        table[i] = AdamWTensor(params[i].data_ptr(), grads[i].data_ptr(), ms[i].data_ptr(), vs[i].data_ptr(),
                               outs[i].data_ptr(), numel, int(steps[i]))
    cfg = AdamWConfig(lr, beta1, beta2, eps, weight_decay)
    if grad_scale is not None and n:
        _expect(grad_scale, "grad_scale", (1,), torch.float32, params[0].device)
        _launch(params[0], lib().mc_adamw_scaled_step, ctypes.byref(cfg), table, n, grad_scale.data_ptr())
        return outs
    stream = _stream(params[0]) if n else None
    check(lib().mc_adamw_step(ctypes.byref(cfg), table, n, stream))
    return outs


def dropout_mask(seed, p, rows, rank):
    """Host-generated keep-mask (uint8 [rows, rank]) as a CPU torch tensor."""
    m = torch.empty(rows, rank, dtype=torch.uint8)
    check(lib().mc_dropout_mask(int(seed), float(p), int(rows), int(rank), ctypes.c_void_p(m.data_ptr())))
    return m
