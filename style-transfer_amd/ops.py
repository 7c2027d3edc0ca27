"""Tensor-level entry points: torch device tensors in, HIP kernels enqueued on the current stream.

`compute` defaults to "f16" (SID_COMPUTE_F16QK: half-precision query/key operands, bf16 probabilities and
values), the arithmetic that holds the path's 2e-2 bar at feature-sized logits; "bf16" and "fp32" select
the other two.  The long-sequence kernels refuse "f16" for logit scales outside [2^-10, 2^10] / log2(e)
(SID_EINVAL); style_transfer_amd.attention.resolve_compute picks "bf16" for such calls.

PyTorch is used for device memory and streams only; all arithmetic of the path happens in
libsid.so.  Every function raises if the library is missing or rejects the call.
"""
import contextlib
import functools
import threading

import torch

from . import lib as _lib

_workspaces = {}

# Held by a thread while it captures a HIP graph (graphed.GraphedUNet) and, in short pieces, by the feature
# loader's worker thread around its GPU calls.  The two must not overlap: with the capturing thread in the
# thread-local capture mode the runtime accepts another thread's allocations and copies during the capture, but
# a blocking copy from pageable memory that races with it fails now and then with "operation not permitted when
# stream is capturing" (measured: once in a few thousand copies), and a failed call invalidates nothing but
# itself, so the loader would lose a file.
capture_lock = threading.RLock()


def _dtype_code(t):
    if t.dtype == torch.float32:
        return _lib.DTYPE_F32
    if t.dtype == torch.bfloat16:
        return _lib.DTYPE_BF16
    raise TypeError("tensors must be float32 or bfloat16, got %s" % t.dtype)


def _compute_code(compute):
    if compute in ("bf16", _lib.COMPUTE_BF16):
        return _lib.COMPUTE_BF16
    if compute in ("fp32", "f32", "f32x3", _lib.COMPUTE_F32X3):
        return _lib.COMPUTE_F32X3
    if compute in ("f16", "f16qk", _lib.COMPUTE_F16QK):
        return _lib.COMPUTE_F16QK
    raise ValueError("compute must be 'bf16', 'f16' or 'fp32', got %r" % (compute,))


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)       # what current_stream(device).cuda_stream reads, 2 us sooner


_HERE = contextlib.nullcontext()


def _on(device):
    """The device context of a launch: nothing to switch (and 1.4 us less) when `device` is the current one."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


_retired = []        # superseded workspaces stay alive: a captured HIP graph may hold their address


def _workspace(device, nbytes):
    """One growing scratch buffer per (device, stream): calls on one stream run in order, so
    they can share it; allocation happens here, never inside the library.  A HIP graph captured on
    the stream bakes the buffer's address in, so the buffer must not grow during capture (warm up
    eagerly with the largest shape first) and a buffer that is outgrown later is kept, not freed."""
    key = (device.index, _stream(device))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("libsid workspace of %d bytes would have to be allocated during graph capture: run the "
                               "call sequence once eagerly on this stream first" % nbytes)
        if ws is not None:
            _retired.append(ws)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def _call_scratch(device, nbytes):
    """Scratch memory of this call's own, for the entry points whose launches pass partial results through it: calls of two
    threads on one stream, and two graphs captured on one stream and replayed on different ones, never share it (a captured
    call's lies in its graph's memory pool)."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _need_cuda(*ts):
    dev = ts[0].device
    for t in ts:
        if t.device.type != "cuda":
            raise RuntimeError("libsid kernels need tensors in GPU memory (got %s)" % t.device)
        if t.device != dev:
            raise RuntimeError("all tensors must be on the same device")
        if not t.is_contiguous():
            raise RuntimeError("tensors must be contiguous")
    return dev


def injected_attention(x_q, q_cnt, k1, v1, k2, v2, k_cnt, v_cnt, mask_signed, gamma, T, scale,
                       heads, q_self_coef=0.5, compute="f16", out=None, flags=0, static_scratch=False):
    """x_q (B,N,H*d); q_cnt,k*,v* (B*H,N,d); mask_signed (B,N) or (N,) float32 -> (B,N,H*d).
    static_scratch=True goes through sid_injected_attn_fwd_static (pass `out` to keep the call free of
    allocations altogether); calls on one GPU must then not overlap."""
    L = _lib.load()
    B, N, C = x_q.shape
    H = heads
    d = C // H
    ts = (x_q, q_cnt, k1, v1, k2, v2, k_cnt, v_cnt)
    dev = _need_cuda(*ts, mask_signed)
    for t in ts[1:]:
        if tuple(t.shape) != (B * H, N, d):
            raise ValueError("feature tensors must be (B*H, N, d) = %s, got %s" % ((B * H, N, d), tuple(t.shape)))
        if t.dtype != x_q.dtype:
            raise TypeError("all attention tensors must share one dtype")
    if mask_signed.dtype != torch.float32 or mask_signed.numel() != B * N:
        raise ValueError("mask_signed must be float32 with B*N elements")
    dt = _dtype_code(x_q)
    cc = _compute_code(compute)
    if out is None:
        out = torch.empty((B, N, C), dtype=x_q.dtype, device=dev)
    if static_scratch:
        # the entry point that allocates nothing: scratch is the library's static device array
        with torch.cuda.device(dev):
            _lib.check(L.sid_injected_attn_fwd_static(
                x_q.data_ptr(), q_cnt.data_ptr(), k1.data_ptr(), v1.data_ptr(), k2.data_ptr(), v2.data_ptr(),
                k_cnt.data_ptr(), v_cnt.data_ptr(), mask_signed.data_ptr(), out.data_ptr(),
                B, H, N, d, float(gamma), float(q_self_coef), float(T), float(scale), dt, cc, int(flags),
                _stream(dev)))
        return out
    nbytes = L.sid_injected_attn_workspace_bytes(B, H, N, d, cc)
    if nbytes == 0:
        raise _lib.SidError(-22, L.sid_last_error().decode())
    ws = _workspace(dev, nbytes)
    with torch.cuda.device(dev):
        _lib.check(L.sid_injected_attn_fwd(
            x_q.data_ptr(), q_cnt.data_ptr(), k1.data_ptr(), v1.data_ptr(), k2.data_ptr(), v2.data_ptr(),
            k_cnt.data_ptr(), v_cnt.data_ptr(), mask_signed.data_ptr(), out.data_ptr(),
            B, H, N, d, float(gamma), float(q_self_coef), float(T), float(scale), dt, cc, int(flags),
            ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


FLAG_THROUGHPUT = 2      # SID_FLAG_THROUGHPUT: the caller keeps the GPU busy with other streams
FLAG_BLOCK_SKIP = 1      # SID_FLAG_BLOCK_SKIP: drop key blocks whose softmax mass is provably nil


def skip_counts(x_q, heads, compute="f16", flags=FLAG_BLOCK_SKIP, packed=False, T=None, scale=None):
    """The block-skipping counters of the last injected-attention call made on the current stream with this
    shape, mode, flags and entry point: (query groups with a dead style block, content segments reduced to
    their logits, of those redone in full, query groups), or None where the flag has no effect (then the
    call ran as if it were not set).  `packed`: False = injected_attention, True = injected_attention_packed,
    "cached" = injected_attention_cached.  Pass the call's T and scale: the library ignores the flag for
    non-positive or vanishing logit scales, and the counters of such a call are not written.  Synchronises."""
    L = _lib.load()
    B, N, C = x_q.shape
    if T is not None and scale is not None:
        log2e = 1.4426950408889634
        if not (T > 0 and scale > 0 and T * scale * log2e >= 2.0 ** -30 and scale * log2e >= 2.0 ** -30):
            return None
    off = L.sid_injected_attn_skip_counts_offset(B, heads, N, C // heads, _compute_code(compute), int(flags),
                                                 2 if packed == "cached" else int(bool(packed)))
    if off < 0:
        return None
    ws = _workspaces.get((x_q.device.index, _stream(x_q.device)))
    if ws is None or off + 16 > ws.numel():
        raise RuntimeError("no injected-attention call with this shape has run on the current stream")
    return tuple(int(v) for v in ws[off:off + 16].view(torch.int32).cpu())


class PackedKV:
    """The key/value pair of one feature-list entry in the kernels' operand layout (sid_pack_kv): what a
    feature store keeps in HBM instead of the two (B*H, N, d) tensors.  Stands in for BOTH tensors in
    the injected-attention call (pass the same object as k and v)."""

    def __init__(self, image, B, H, N, d, compute):
        self.image, self.B, self.H, self.N, self.d, self.compute = image, B, H, N, d, compute
        self.partial = None     # a content pair may carry its cached content block (ContentPartial)

    @property
    def device(self):
        return self.image.device

    def nbytes(self):
        return self.image.numel()


def pack_kv(k, v, heads, compute="f16"):
    """k, v (B*H, N, d) float32 / bfloat16 -> PackedKV (one launch on the current stream)."""
    L = _lib.load()
    dev = _need_cuda(k, v)
    if k.shape != v.shape or k.dtype != v.dtype or k.dim() != 3 or k.shape[0] % heads:
        raise ValueError("k and v must be two (B*H, N, d) tensors of one dtype")
    BH, N, d = k.shape
    B = BH // heads
    cc = _compute_code(compute)
    nbytes = L.sid_kv_image_bytes(B, heads, N, d, cc)
    if nbytes == 0:
        raise _lib.SidError(-22, L.sid_last_error().decode())
    image = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L.sid_pack_kv(k.data_ptr(), v.data_ptr(), image.data_ptr(), nbytes, B, heads, N, d, _dtype_code(k), cc,
                                 _stream(dev)))
    return PackedKV(image, B, heads, N, d, cc)


def injected_attention_packed(x_q, q_cnt, kv1, kv2, kv_cnt, mask_signed, gamma, T, scale, heads, q_self_coef=0.5,
                              out=None, flags=0):
    """injected_attention with the three key/value pairs pre-packed (PackedKV); same results."""
    L = _lib.load()
    B, N, C = x_q.shape
    H = heads
    d = C // H
    dev = _need_cuda(x_q, q_cnt, mask_signed, kv1.image, kv2.image, kv_cnt.image)
    if tuple(q_cnt.shape) != (B * H, N, d) or q_cnt.dtype != x_q.dtype:
        raise ValueError("q_cnt must be (B*H, N, d) = %s of x_q's dtype" % ((B * H, N, d),))
    cc = kv1.compute
    for kv in (kv1, kv2, kv_cnt):
        if (kv.B, kv.H, kv.N, kv.d, kv.compute) != (B, H, N, d, cc):
            raise ValueError("packed K/V was made for (B,H,N,d,compute) = %s, the call has %s"
                             % ((kv.B, kv.H, kv.N, kv.d, kv.compute), (B, H, N, d, cc)))
    if mask_signed.dtype != torch.float32 or mask_signed.numel() != B * N:
        raise ValueError("mask_signed must be float32 with B*N elements")
    if out is None:
        out = torch.empty((B, N, C), dtype=x_q.dtype, device=dev)
    nbytes = L.sid_injected_attn_packed_workspace_bytes(B, H, N, d, cc)
    if nbytes == 0:
        raise _lib.SidError(-22, L.sid_last_error().decode())
    ws = _workspace(dev, nbytes)
    with torch.cuda.device(dev):
        _lib.check(L.sid_injected_attn_fwd_packed(
            x_q.data_ptr(), q_cnt.data_ptr(), kv1.image.data_ptr(), kv2.image.data_ptr(), kv_cnt.image.data_ptr(),
            mask_signed.data_ptr(), out.data_ptr(), B, H, N, d, float(gamma), float(q_self_coef), float(T), float(scale),
            _dtype_code(x_q), cc, int(flags), ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


class ContentPartial:
    """The content block of the injected attention for one (timestep, layer) of a content feature file
    (sid_content_partial): per (head, row) the block's normalised output row, softmax reference and row
    sum, and the q_cnt.k_cnt extremes the mask bias needs.  It depends on q_cnt, k_cnt, v_cnt and `scale`
    only, so one content image stylised with several style pairs computes it once."""

    def __init__(self, data, B, H, N, d, compute, scale, q_ptr):
        self.data, self.B, self.H, self.N, self.d, self.compute, self.scale = data, B, H, N, d, compute, scale
        self.q_ptr = q_ptr          # address of the q_cnt tensor it was made from (calls check they pass the same one)

    @property
    def device(self):
        return self.data.device

    def nbytes(self):
        return self.data.numel()


def content_partial(q_cnt, kv_cnt, scale, heads):
    """q_cnt (B*H, N, d) and the content pair's PackedKV -> ContentPartial (two launches on the current stream)."""
    L = _lib.load()
    dev = _need_cuda(q_cnt, kv_cnt.image)
    B, H, N, d, cc = kv_cnt.B, kv_cnt.H, kv_cnt.N, kv_cnt.d, kv_cnt.compute
    if H != heads or tuple(q_cnt.shape) != (B * H, N, d):
        raise ValueError("q_cnt must be (B*H, N, d) = %s, got %s" % ((B * H, N, d), tuple(q_cnt.shape)))
    nbytes = L.sid_content_partial_bytes(B, H, N, d, cc)
    wbytes = L.sid_content_partial_workspace_bytes(B, H, N, d, cc)
    if nbytes == 0 or wbytes == 0:
        raise _lib.SidError(-22, L.sid_last_error().decode())
    data = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    ws = _workspace(dev, wbytes)
    with torch.cuda.device(dev):
        _lib.check(L.sid_content_partial(q_cnt.data_ptr(), kv_cnt.image.data_ptr(), data.data_ptr(), nbytes, B, H, N, d,
                                         float(scale), _dtype_code(q_cnt), cc, ws.data_ptr(), ws.numel(), _stream(dev)))
    return ContentPartial(data, B, H, N, d, cc, float(scale), q_cnt.data_ptr())


def content_partials(jobs, heads, streams=4):
    """ContentPartial of every (q_cnt, PackedKV, scale) in `jobs`, in order.  One call is one run per (head,
    query group), 64 workgroups at SD-v1 sizes, a quarter of the GPU, so the calls go round-robin over
    `streams` side streams (each with its own workspace) and the current stream waits for all of them."""
    if not jobs:
        return []
    dev = jobs[0][0].device
    cur = torch.cuda.current_stream(dev)
    side = [torch.cuda.Stream(device=dev) for _ in range(max(1, min(streams, len(jobs))))]
    out = []
    for st in side:
        st.wait_stream(cur)
    for i, (q_cnt, kv, scale) in enumerate(jobs):
        with torch.cuda.stream(side[i % len(side)]):
            out.append(content_partial(q_cnt, kv, scale, heads))
    for st in side:
        cur.wait_stream(st)
    for p in out:                       # made on a side stream, used on this one from here on
        p.data.record_stream(cur)
    return out


def injected_attention_cached(x_q, q_cnt, kv1, kv2, partial, mask_signed, gamma, T, scale, heads, q_self_coef=0.5,
                              out=None, flags=0):
    """injected_attention_packed with the content pair replaced by its ContentPartial: only the two style
    blocks are computed.  `scale` and `q_cnt` must be the ones the partial was made with."""
    L = _lib.load()
    B, N, C = x_q.shape
    H = heads
    d = C // H
    dev = _need_cuda(x_q, q_cnt, mask_signed, kv1.image, kv2.image, partial.data)
    if tuple(q_cnt.shape) != (B * H, N, d) or q_cnt.dtype != x_q.dtype:
        raise ValueError("q_cnt must be (B*H, N, d) = %s of x_q's dtype" % ((B * H, N, d),))
    cc = kv1.compute
    for kv in (kv1, kv2, partial):
        if (kv.B, kv.H, kv.N, kv.d, kv.compute) != (B, H, N, d, cc):
            raise ValueError("packed K/V or content partial was made for (B,H,N,d,compute) = %s, the call has %s"
                             % ((kv.B, kv.H, kv.N, kv.d, kv.compute), (B, H, N, d, cc)))
    if partial.scale != float(scale):
        raise ValueError("the content partial was made with scale %r, the call has %r" % (partial.scale, float(scale)))
    if partial.q_ptr != q_cnt.data_ptr():
        raise ValueError("the content partial was made from another q_cnt tensor")
    if mask_signed.dtype != torch.float32 or mask_signed.numel() != B * N:
        raise ValueError("mask_signed must be float32 with B*N elements")
    if out is None:
        out = torch.empty((B, N, C), dtype=x_q.dtype, device=dev)
    nbytes = L.sid_injected_attn_cached_workspace_bytes(B, H, N, d, cc)
    if nbytes == 0:
        raise _lib.SidError(-22, L.sid_last_error().decode())
    ws = _workspace(dev, nbytes)
    with torch.cuda.device(dev):
        _lib.check(L.sid_injected_attn_fwd_cached(
            x_q.data_ptr(), q_cnt.data_ptr(), kv1.image.data_ptr(), kv2.image.data_ptr(), partial.data.data_ptr(),
            mask_signed.data_ptr(), out.data_ptr(), B, H, N, d, float(gamma), float(q_self_coef), float(T), float(scale),
            _dtype_code(x_q), cc, int(flags), ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


def plain_attention(q, k, v, logit_scale, heads, q_layout="bnhd", kv_layout="bnhd", compute="f16", out=None, flags=0):
    """softmax((q k^T) * logit_scale) v.  Layout 'bnhd': (B,N,H*d); 'bhnd': (B*H,N,d).
    Returns (B, Nq, H*d)."""
    L = _lib.load()
    H = heads
    lay = {"bnhd": _lib.LAYOUT_BNHD, "bhnd": _lib.LAYOUT_BHND}
    dev = _need_cuda(q, k, v)

    def dims(t, layout):
        if layout == "bnhd":
            b, n, c = t.shape
            return b, n, c // H
        bh, n, d_ = t.shape
        return bh // H, n, d_

    B, Nq, d = dims(q, q_layout)
    Bk, Nk, dk = dims(k, kv_layout)
    if (Bk, dk) != (B, d) or tuple(v.shape) != tuple(k.shape):
        raise ValueError("q/k/v shapes disagree: %s %s %s" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k, v must share one dtype")
    dt = _dtype_code(q)
    cc = _compute_code(compute)
    if out is None:
        out = torch.empty((B, Nq, H * d), dtype=q.dtype, device=dev)
    nbytes = L.sid_plain_attn_workspace_bytes(B, H, Nq, Nk, d, cc)
    if nbytes == 0:
        raise _lib.SidError(-22, L.sid_last_error().decode())
    ws = _workspace(dev, nbytes)
    with torch.cuda.device(dev):
        _lib.check(L.sid_plain_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, Nq, Nk, d,
                                        float(logit_scale), lay[q_layout], lay[kv_layout], dt, cc, int(flags),
                                        ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


def mask_downsample(mask, out_h, out_w, ch=1.0):
    """(Hin, Win) float32 mask in [0,1] on the GPU -> signed (out_h*out_w,) float32."""
    L = _lib.load()
    dev = _need_cuda(mask)
    if mask.dtype != torch.float32 or mask.dim() != 2:
        raise ValueError("mask must be a 2-D float32 tensor")
    out = torch.empty(out_h * out_w, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L.sid_mask_downsample(mask.data_ptr(), mask.shape[0], mask.shape[1], out_h, out_w, float(ch),
                                         out.data_ptr(), _stream(dev)))
    return out


def hf_filter(h_cnt, ratio=0.5, skip=None, h=None, out=None):
    """HF(h_cnt), or skip + h + HF(h_cnt) when skip and h are given.  (B,C,H,W) tensors."""
    L = _lib.load()
    ts = [h_cnt] + ([skip, h] if skip is not None else [])
    dev = _need_cuda(*ts)
    if (skip is None) != (h is None):
        raise ValueError("skip and h must be given together")
    for t in ts:
        if t.shape != h_cnt.shape or t.dtype != h_cnt.dtype:
            raise ValueError("skip, h and h_cnt must share shape and dtype")
    B, C, Hh, Ww = h_cnt.shape
    radius = int(min(Hh, Ww) * ratio)          # high_frequency_final.py:18, in double like the reference
    if out is None:
        out = torch.empty_like(h_cnt)
    with torch.cuda.device(dev):
        _lib.check(L.sid_hf_filter_radius(h_cnt.data_ptr(), skip.data_ptr() if skip is not None else None,
                                          h.data_ptr() if h is not None else None, out.data_ptr(),
                                          B, C, Hh, Ww, radius, _dtype_code(h_cnt), _stream(dev)))
    return out


def residual_sum(skip, h, hf, out=None):
    """(skip + h) + hf: the patched ResBlock sum with HF(h_cnt) filtered earlier (hf_filter without skip / h);
    the same bits as the fused hf_filter(h_cnt, ratio, skip, h)."""
    L = _lib.load()
    dev = _need_cuda(skip, h, hf)
    for t in (h, hf):
        if t.shape != skip.shape or t.dtype != skip.dtype:
            raise ValueError("skip, h and hf must share shape and dtype")
    if out is None:
        out = torch.empty_like(skip)
    with torch.cuda.device(dev):
        _lib.check(L.sid_residual_sum(skip.data_ptr(), h.data_ptr(), hf.data_ptr(), out.data_ptr(), skip.numel(),
                                      _dtype_code(skip), _stream(dev)))
    return out


def masked_adain(cnt, sty_char, sty_back=None, mask=None, out=None):
    """m * adain(cnt, sty_char) + (1 - m) * adain(cnt, sty_back) with m the raw (Hin, Win) float32 mask
    resized bilinearly to the latent; with sty_back and mask None: adain(cnt, sty_char).  (B,C,H,W)."""
    L = _lib.load()
    ts = [cnt, sty_char] + ([sty_back] if sty_back is not None else [])
    dev = _need_cuda(*ts)
    if (sty_back is None) != (mask is None):
        raise ValueError("sty_back and mask go together")
    for t in ts:
        if tuple(t.shape) != tuple(cnt.shape) or t.dtype != cnt.dtype or t.dim() != 4:
            raise ValueError("latents must share one (B,C,H,W) shape and dtype")
    if mask is not None:
        _need_cuda(mask)
        if mask.dtype != torch.float32 or mask.dim() != 2 or mask.device != dev:
            raise ValueError("mask must be a 2-D float32 tensor on the latents' device")
    B, C, H, W = cnt.shape
    if out is None:
        out = torch.empty_like(cnt)
    with torch.cuda.device(dev):
        _lib.check(L.sid_masked_adain(cnt.data_ptr(), sty_char.data_ptr(),
                                      sty_back.data_ptr() if sty_back is not None else None,
                                      mask.data_ptr() if mask is not None else None,
                                      mask.shape[0] if mask is not None else 0, mask.shape[1] if mask is not None else 0,
                                      out.data_ptr(), B, C, H, W, _dtype_code(cnt), _stream(dev)))
    return out


# ------------------------------------------------------------------------------------------------
# Key/value cache in 8 bits
# ------------------------------------------------------------------------------------------------
_DTYPES3 = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_KV_FORMATS = {torch.int8: _lib.KV_INT8, torch.float8_e4m3fn: _lib.KV_E4M3}


def _need_device(dev, *ts):
    """Every tensor in the memory of the one GPU `dev` (strides are the caller's matter)."""
    if dev.type != "cuda":
        raise RuntimeError("libsid kernels need tensors in GPU memory (got %s)" % dev)
    for t in ts:
        if t.device != dev:
            raise RuntimeError("all tensors must be on the same device (%s and %s)" % (dev, t.device))


def _rows16(t):
    """`t` (..., d) with d contiguous and every row on a 16-byte boundary (itself, or a copy), its address, its strides."""
    st, ptr = t.stride(), t.data_ptr()
    steps = st[0] | st[1] | st[-2]                       # of three or four dimensions
    if st[-1] != 1 or (ptr | steps * t.element_size()) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, t.data_ptr(), t.stride()
    return t, ptr, st


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(name, *shape):
    """What a call of this shape needs, from the library (which refuses the shape with 0)."""
    L = _lib.load()
    n = getattr(L, name)(*shape)
    if n == 0:
        raise _lib.SidError(-22, L.sid_last_error().decode())
    return n


class QuantKV:
    """Keys and values of B sequences in 8 bits: codes (B, H, S, d) as torch.int8 or torch.float8_e4m3fn and one float32
    scale per row (B, H, S); a code stands for code * scale.  Made empty by kv_cache(), filled by kv_cache_write(),
    read by kv_cache_read() and, without becoming 16-bit tensors in memory first, by shared_prefix_attention()."""

    def __init__(self, k_codes, k_scale, v_codes, v_scale):
        fmt, shape, dev = _KV_FORMATS.get(k_codes.dtype), k_codes.shape, k_codes.device
        if fmt is None or v_codes.dtype != k_codes.dtype:
            raise TypeError("codes must be int8 or float8_e4m3fn, keys and values alike, got %s and %s" % (k_codes.dtype, v_codes.dtype))
        if len(shape) != 4 or v_codes.shape != shape:
            raise ValueError("codes must be two (B, H, S, d) tensors, got %s and %s" % (tuple(shape), tuple(v_codes.shape)))
        if not k_scale.dtype == v_scale.dtype == torch.float32 or not k_scale.shape == v_scale.shape == shape[:3]:
            raise ValueError("scales must be float32 (B, H, S) = %s" % (tuple(shape[:3]),))
        if not (k_codes.is_contiguous() and v_codes.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise RuntimeError("tensors must be contiguous")
        if not v_codes.device == k_scale.device == v_scale.device == dev:
            raise RuntimeError("all tensors must be on the same device")
        self.k_codes, self.k_scale, self.v_codes, self.v_scale = k_codes, k_scale, v_codes, v_scale
        self.B, self.H, self.S, self.d = shape
        self.device, self.fmt = dev, fmt

    def tensors(self):
        return self.k_codes, self.k_scale, self.v_codes, self.v_scale

    def nbytes(self):
        return 2 * (self.k_codes.numel() + 4 * self.k_scale.numel())

    def _source(self):
        d, S = self.d, self.S
        Sd, HS = S * d, self.H * S
        return _lib.kv_source(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                              HS * d, Sd, d, HS * d, Sd, d, HS, S, self.fmt)


def kv_cache(batch, heads, length, head_dim, fmt="int8", device="cuda"):
    """An empty QuantKV (every position reads as zeros): `length` positions for each of `batch` sequences.  fmt "int8"
    (rows of even magnitude: half the error of e4m3 on normally distributed features) or "e4m3" (rows with a few
    large values: the small ones keep their relative precision)."""
    dt = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}.get(fmt)
    if dt is None:
        raise ValueError("cache format must be 'int8' or 'e4m3', got %r" % (fmt,))
    if head_dim % 8 or not 8 <= head_dim <= 256:
        raise ValueError("head_dim must be a multiple of 8 in [8, 256], got %d" % head_dim)
    shape = (batch, heads, length, head_dim)
    codes = [torch.zeros(shape, dtype=torch.uint8, device=device).view(dt) for _ in range(2)]
    scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
    return QuantKV(codes[0], scales[0], codes[1], scales[1])


def _positions(start, B, dev):
    if isinstance(start, int):
        return torch.full((B,), start, dtype=torch.int32, device=dev)
    if start.dtype != torch.int32 or tuple(start.shape) != (B,) or not start.is_contiguous():
        raise ValueError("positions and lengths must be contiguous int32 (B,) = (%d,), got %s %s" % (B, start.dtype, tuple(start.shape)))
    return start


def kv_cache_write(cache, k, v, start=0, length=None):
    """Quantise k, v (B, H, n, d) (float32, bfloat16 or float16; any strides with d contiguous) into positions start[b] + i of
    sequence b.  start: an int, or an int32 (B,) tensor on the device (nothing is read back, so a decoding step can be
    captured in a HIP graph).  length: int32 (B,) tensor, rows i >= length[b] are padding and not written; None: all n.
    Positions outside the cache are skipped; everything else in it stays as it was.  One launch, and a second that fills a
    tensor with an int start."""
    L = _lib.load()
    dev = cache.device
    if k.shape != v.shape or k.dtype != v.dtype or k.dim() != 4:
        raise ValueError("k and v must be two (B, H, n, d) tensors of one dtype")
    B, H, n, d = k.shape
    if (B, H, d) != (cache.B, cache.H, cache.d):
        raise ValueError("the cache holds (B, H, d) = %s, the call has %s" % ((cache.B, cache.H, cache.d), (B, H, d)))
    if k.dtype not in _DTYPES3:
        raise TypeError("tensors must be float32, bfloat16 or float16, got %s" % k.dtype)
    start = _positions(start, B, dev)
    if length is not None:
        length = _positions(length, B, dev)
        _need_device(dev, length)
    _need_device(dev, k, v, start)
    if cache.k_codes.numel() == 0:               # no position to write to
        return
    k, kp, ks = _rows16(k)
    v, vp, vs = _rows16(v)
    with _on(dev):
        _lib.check(L.sid_kv_cache_write(kp, vp, _lib.strides3(*ks[:3]), _lib.strides3(*vs[:3]),
                                        cache.k_codes.data_ptr(), cache.v_codes.data_ptr(), cache.k_scale.data_ptr(),
                                        cache.v_scale.data_ptr(), start.data_ptr(), None if length is None else length.data_ptr(),
                                        B, H, n, cache.S, d, _DTYPES3[k.dtype], cache.fmt, _stream(dev)))


def kv_cache_read(cache, start, n, dtype=torch.bfloat16):
    """The n positions from start[b] on (int, or int32 (B,) tensor on the device) as numbers: k, v (B, H, n, d) in `dtype`.
    Positions outside the cache give zeros.  One launch, and a second that fills a tensor with an int start."""
    L = _lib.load()
    dev = cache.device
    if dtype not in _DTYPES3:
        raise TypeError("tensors must be float32, bfloat16 or float16, got %s" % dtype)
    if n < 0:
        raise ValueError("n must not be negative")
    start = _positions(start, cache.B, dev)
    _need_device(dev, start)
    shape = (cache.B, cache.H, n, cache.d)
    if cache.k_codes.numel() == 0:               # every position is outside
        return torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev)
    k, v = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
    with _on(dev):
        _lib.check(L.sid_kv_cache_read(cache.k_codes.data_ptr(), cache.v_codes.data_ptr(), cache.k_scale.data_ptr(),
                                       cache.v_scale.data_ptr(), k.data_ptr(), v.data_ptr(), start.data_ptr(),
                                       cache.B, cache.H, n, cache.S, cache.d, _DTYPES3[dtype], cache.fmt, _stream(dev)))
    return k, v


# ------------------------------------------------------------------------------------------------
# Attention of a batch that shares a prefix
# ------------------------------------------------------------------------------------------------
def _pair_source(k, v, dtype, what):
    """(k, v) tensors (B, H, keys, d), or (H, keys, d) for a prefix -> (sid_kv_source, tensors to keep alive)."""
    if v.shape != k.shape or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("%s: keys and values must be alike and %s, got %s %s and %s %s"
                         % (what, dtype, tuple(k.shape), k.dtype, tuple(v.shape), v.dtype))
    k, kp, ks = _rows16(k)
    v, vp, vs = _rows16(v)
    if len(ks) == 3:
        return _lib.kv_source(kp, vp, 0, 0, 0, ks[0], ks[1], 0, vs[0], vs[1], 0, 0, _lib.KV_NONE), (k, v)
    return _lib.kv_source(kp, vp, 0, 0, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], 0, 0, _lib.KV_NONE), (k, v)


def shared_prefix_attention(q, prefix=None, own=None, own_len=None, causal=False, scale=None, prefix_len=None, out=None):
    """Attention of a batch whose sequences share a prefix of keys and values, under one softmax with their own keys.

    q (B, Hq, n, d) bfloat16 or float16, any strides with d contiguous; n = 1 for a decoding step.
    prefix: (k, v) of shape (Hkv, P, d), one copy for the whole batch, or a QuantKV with B = 1; None: no prefix.  (Parts in
        8 bits of head_dim 8 are copied to rows of 16 in every call.)
        prefix_len: only its first keys (an int); None: all.
    own: (k, v) of shape (B, Hkv, S, d), or a QuantKV with the batch's B; None: none.
        own_len: int32 (B,) tensor on the device, how many of its own keys each sequence has (clamped to [0, S]).
        causal: query i of a sequence sees its own keys j <= own_len - n + i.
    Hq must be a multiple of Hkv (query head h reads key/value head h // (Hq // Hkv)).  scale: d ** -0.5 if None.
    -> (B, n, Hq*d) of q's dtype.  A query that sees no key gives zeros.  Forward only: where q or a 16-bit key or value
    requires a gradient, a backward pass through the result raises an error, and `out` is refused."""
    if torch.is_grad_enabled():
        tracked, prefix = _tracked(prefix)
        tracked_own, own = _tracked(own)
        if tracked or tracked_own or q.requires_grad:
            if out is not None:
                raise RuntimeError("shared_prefix_attention: out= takes no inputs that require a gradient")
            inputs = [t for p in ((q,), prefix, own) if p is not None and not isinstance(p, QuantKV) for t in p]
            return _SharedPrefixForward.apply(lambda: _shared_prefix(q, prefix, own, own_len, causal, scale, prefix_len, None), *inputs)
    return _shared_prefix(q, prefix, own, own_len, causal, scale, prefix_len, out)


def _tracked(part):
    """Whether a key or value of the part requires a gradient; the part, its pair as a tuple."""
    if part is None or isinstance(part, QuantKV):
        return False, part
    k, v = part = tuple(part)
    return k.requires_grad or v.requires_grad, part


class _SharedPrefixForward(torch.autograd.Function):
    """The call's place in an autograd graph: without it the result would be cut off from q, keys and values silently."""

    @staticmethod
    def forward(ctx, call, *tracked):
        return call()

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("shared_prefix_attention is forward only: it has no gradient for q, keys and values")


def _pad8(t):
    return torch.nn.functional.pad(t, (0, 8))


def _sixteen(part):
    """A part of head_dim 8 as one of 16, zeros behind every row."""
    if part is None:
        return None
    if isinstance(part, QuantKV):
        k, v = (_pad8(c.view(torch.uint8)).view(c.dtype) for c in (part.k_codes, part.v_codes))
        return QuantKV(k, part.k_scale, v, part.v_scale)
    return tuple(_pad8(t) for t in part)


def _checked_out(out, shape, dtype, dev):
    if out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError("out must be a contiguous %s %s on %s" % (tuple(shape), dtype, dev))
    return out


def _shared_prefix(q, prefix, own, own_len, causal, scale, prefix_len, out):
    L = _lib.load()
    dev = q.device
    if q.dim() != 4:
        raise ValueError("q must be (B, Hq, n, d), got %s" % (tuple(q.shape),))
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("q must be bfloat16 or float16, got %s" % q.dtype)
    B, Hq, n, d = q.shape
    _need_device(dev)
    if d == 8 and (isinstance(prefix, QuantKV) or isinstance(own, QuantKV)):
        # the kernel reads codes sixteen at a time: eight zeros behind every row add nothing to a product
        y = _shared_prefix(_pad8(q), _sixteen(prefix), _sixteen(own), own_len, causal, d ** -0.5 if scale is None else scale, prefix_len, None)
        y = y.view(B, n, Hq, 16)[..., :8].reshape(B, n, Hq * 8)
        return y if out is None else _checked_out(out, y.shape, y.dtype, dev).copy_(y)
    P = S = 0
    Hp = Ho = None
    src_p = src_o = alive = None
    fmt_p = fmt_o = _lib.KV_NONE
    if prefix is not None:
        if isinstance(prefix, QuantKV):
            if prefix.B != 1 or prefix.d != d:
                raise ValueError("prefix: the cache holds (B, d) = %s, the call needs %s" % ((prefix.B, prefix.d), (1, d)))
            _need_device(dev, prefix.k_codes)
            Hp, P, src_p, fmt_p = prefix.H, prefix.S, prefix._source(), prefix.fmt
        else:
            k, v = prefix
            if k.dim() != 3 or k.shape[2] != d:
                raise ValueError("prefix: keys must be (H, P, %d), got %s" % (d, tuple(k.shape)))
            _need_device(dev, k, v)
            Hp, P = k.shape[:2]
            src_p, alive = _pair_source(k, v, q.dtype, "prefix")
    if own is not None:
        if isinstance(own, QuantKV):
            if own.B != B or own.d != d:
                raise ValueError("own part: the cache holds (B, d) = %s, the call needs %s" % ((own.B, own.d), (B, d)))
            _need_device(dev, own.k_codes)
            Ho, S, src_o, fmt_o = own.H, own.S, own._source(), own.fmt
        else:
            k, v = own
            if k.dim() != 4 or k.shape[0] != B or k.shape[3] != d:
                raise ValueError("own part: keys must be (%d, H, S, %d), got %s" % (B, d, tuple(k.shape)))
            _need_device(dev, k, v)
            Ho, S = k.shape[1:3]
            src_o, alive_o = _pair_source(k, v, q.dtype, "own part")
            alive = (alive, alive_o)
    Hkv = Hp if Ho is None else Ho
    if Hkv is None:
        raise ValueError("neither a prefix nor own keys")
    if Hp not in (None, Hkv):
        raise ValueError("prefix and own part differ in heads: %d and %d" % (Hp, Ho))
    if prefix_len is not None:
        if not 0 <= prefix_len <= P:
            raise ValueError("prefix_len %d is outside [0, %d]" % (prefix_len, P))
        P = int(prefix_len)
    if own_len is not None:
        own_len = _positions(own_len, B, dev)
        _need_device(dev, own_len)
    q, qp, qs = _rows16(q)
    out = torch.empty((B, n, Hq * d), dtype=q.dtype, device=dev) if out is None else _checked_out(out, (B, n, Hq * d), q.dtype, dev)
    ws = _call_scratch(dev, _scratch_bytes("sid_shared_attn_workspace_bytes", B, Hq, Hkv, n, d, P, S,
                                         int(P and S and fmt_p != fmt_o)))
    with _on(dev):
        _lib.check(L.sid_shared_attn_fwd(
            qp, _lib.strides3(qs[0], qs[1], qs[2]), src_p, src_o, None if own_len is None else own_len.data_ptr(),
            out.data_ptr(), B, Hq, Hkv, n, d, P, S, float(d ** -0.5 if scale is None else scale), int(causal),
            _DTYPES3[q.dtype], ws.data_ptr(), ws.numel(), _stream(dev)))
    return out


# ------------------------------------------------------------------------------------------------
# Group normalisation with an activation, channels last
# ------------------------------------------------------------------------------------------------
_ACTS = {"none": _lib.ACT_NONE, "silu": _lib.ACT_SILU}


def _norm_shape(x, groups):
    """(B, N, C) of a channels-last tensor: (B, C, H, W) in channels-last memory, or (B, N, C) contiguous."""
    if x.dim() == 4:
        if not x.is_contiguous(memory_format=torch.channels_last):
            raise ValueError("a (B, C, H, W) tensor must be in channels-last memory (x.contiguous(memory_format=torch.channels_last))")
        B, C, H, W = x.shape
        return B, H * W, C
    if x.dim() == 3:
        if not x.is_contiguous():
            raise ValueError("a (B, N, C) tensor must be contiguous")
        return tuple(x.shape)
    raise ValueError("x must be (B, C, H, W) in channels-last memory or (B, N, C), got %s" % (tuple(x.shape),))


def _norm_forward(x, groups, weight, bias, eps, act, keep):
    """-> y and, for a backward pass (`keep`), a tensor that holds the float32 mean and rstd (2, B, groups) from a byte
    offset on, that offset and the sizes of the call."""
    L = _lib.load()
    dev = x.device
    B, N, C = _norm_shape(x, groups)
    dt = _DTYPES3.get(x.dtype)
    if dt is None:
        raise TypeError("x must be float32, bfloat16 or float16, got %s" % x.dtype)
    wp = bp = None
    if weight is not None:
        _norm_param(dev, weight, C)
        wp = weight.data_ptr()
    if bias is not None:
        _norm_param(dev, bias, C)
        bp = bias.data_ptr()
    _need_device(dev)
    y = torch.empty_like(x)
    need = _scratch_bytes("sid_group_norm_workspace_bytes", B, N, C, groups, dt, 0)
    half, at = 4 * B * groups, (need + 3) // 4 * 4
    if keep and need > 65536:                # what the backward pass keeps alive is the statistics alone
        ws, stats, at = _call_scratch(dev, need), _call_scratch(dev, 2 * half), 0
    else:                                    # one allocation for both: the scratch memory first, it wants the alignment
        ws = stats = _call_scratch(dev, at + 2 * half)
    sp = stats.data_ptr() + at
    act = _ACTS[act]
    with _on(dev):
        _lib.check(L.sid_group_norm_act_fwd(x.data_ptr(), wp, bp, y.data_ptr(), sp, sp + half, B, N, C, groups, eps, act, dt,
                                            ws.data_ptr(), need, _stream(dev)))
    return y, stats, (at, B, N, C, groups, act, dt)


def _norm_param(dev, t, C):
    if t.shape != (C,) or t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError("weight and bias must be contiguous float32 (C,) = (%d,)" % C)
    _need_device(dev, t)


def _norm_backward(ctx, dy):
    """Runs on autograd's own thread, which wakes up for it on a core that may be slow: nothing is decided here that the
    forward pass knew."""
    x, weight, bias, stats = ctx.saved_tensors
    at, B, N, C, G, act, dt = ctx.call
    dev = x.device
    if dy.dtype != x.dtype or dy.stride() != x.stride():
        dy = dy.to(x.dtype).contiguous(memory_format=torch.channels_last if x.dim() == 4 else torch.contiguous_format)
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dx = torch.empty_like(x) if need_x else None
    dw = torch.empty_like(weight) if need_w else None
    db = torch.empty_like(bias) if need_b else None
    need = _scratch_bytes("sid_group_norm_workspace_bytes", B, N, C, G, dt, 1)
    ws = _call_scratch(dev, need)
    sp = stats.data_ptr() + at
    with _on(dev):
        _lib.check(_lib.load().sid_group_norm_act_bwd(
            dy.data_ptr(), x.data_ptr(), None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(),
            sp, sp + 4 * B * G, dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None, db.data_ptr() if need_b else None,
            B, N, C, G, act, dt, ws.data_ptr(), need, _stream(dev)))
    return dx, dw, db, None, None, None


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, stats, ctx.call = _norm_forward(x, groups, weight, bias, eps, act, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():          # create_graph: the result refuses a second derivative
            return _norm_backward_once(ctx, dy)
        return _norm_backward(ctx, dy)


_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="silu"):
    """act(group_norm(x) * weight + bias) over channels-last tensors, differentiable in x, weight and bias.

    x (B, C, H, W) in channels-last memory, or tokens (B, N, C) contiguous; float32, bfloat16 or float16.  weight, bias:
    float32 (C,) or None (other float types are cast, with gradients).  act: "silu" or "none".  Statistics, gradients of
    weight and bias and all arithmetic are float32; y has x's dtype and memory order.  Needs at least one value.  A training
    step can be captured; as with torch's own operators, only while no eager graph of the same leaves is alive."""
    if act not in _ACTS:
        raise ValueError("act must be 'silu' or 'none', got %r" % (act,))
    eps = float(eps)
    if weight is not None and weight.dtype != torch.float32:
        weight = weight.float()
    if bias is not None and bias.dtype != torch.float32:
        bias = bias.float()
    if torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        return _GroupNormAct.apply(x, weight, bias, groups, eps, act)
    return _norm_forward(x, groups, weight, bias, eps, act, False)[0]
