"""Python mirror of the reference's hot-path call surface (``namespace hip`` in
engine/kernels/gemv.h, gemm.h and fn.h), over the C ABI of libhipster_qmm.so.

Same function names, argument meaning and output layout as the reference; torch CUDA tensors stand
in for the device pointers (torch is only the device-memory and stream plumbing here).  Errors that
the reference turns into ``abort()`` raise ``QmmError`` instead.  Every call launches on the current
torch stream unless ``stream`` is given.
"""
import ctypes

import torch

from . import _lib
from ._lib import KVMX, XMX, XQ8, XQ8K, Attn, Gate, GemvSeg, MoeSegs, MoeTile, QmmError, Rope, RouteRule, Seqs, check  # noqa: F401

WFmt = type("WFmt", (), {"Q4_K": _lib.QMM_Q4_K, "Q5_K": _lib.QMM_Q5_K, "IQ4_XS": _lib.QMM_IQ4_XS,
                         "Q6_K_SOA": _lib.QMM_Q6_K_SOA, "Q8_0_SOA": _lib.QMM_Q8_0_SOA,
                         "Q5_1_SOA": _lib.QMM_Q5_1_SOA, "Q6_K": _lib.QMM_Q6_K})


def _p(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream(stream):
    s = torch.cuda.current_stream() if stream is None else stream
    return ctypes.c_void_p(s.cuda_stream)


def _dev(t, dtype=None, name="tensor"):
    if t is None or not t.is_cuda:
        raise QmmError(f"{name} must be a CUDA tensor")
    if dtype is not None and t.dtype != dtype:
        raise QmmError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise QmmError(f"{name} must be contiguous")
    return t


class XQ8Buf:
    """Device buffers of XQ8 (gemv.h:8): q [ncol][K] int8, d/s [ncol][K/32] f32, optional ds."""

    def __init__(self, ncol, K, device="cuda", with_ds=False):
        self.ncol, self.K = ncol, K
        self.q = torch.zeros((ncol, K), dtype=torch.int8, device=device)
        self.d = torch.zeros((ncol, K // 32), dtype=torch.float32, device=device)
        self.s = torch.zeros((ncol, K // 32), dtype=torch.float32, device=device)
        self.ds = torch.zeros((ncol, K // 32, 2), dtype=torch.float32, device=device) if with_ds else None

    def c(self):
        return XQ8(self.q.data_ptr(), self.d.data_ptr(), self.s.data_ptr(), 0 if self.ds is None else self.ds.data_ptr())


class XQ8KBuf:
    """Device buffers of XQ8K (gemv.h:33): q [ncol][K] int8, d [K/256][16] f32, bs [K/256][16][8] int16."""

    def __init__(self, ncol, K, device="cuda"):
        self.ncol, self.K = ncol, K
        self.q = torch.zeros((ncol, K), dtype=torch.int8, device=device)
        self.d = torch.zeros((K // 256, 16), dtype=torch.float32, device=device)
        self.bs = torch.zeros((K // 256, 16, 8), dtype=torch.int16, device=device)

    def c(self):
        return XQ8K(self.q.data_ptr(), self.d.data_ptr(), self.bs.data_ptr())


def wfmt_row_bytes(fmt, K):
    return _lib.lib().qmm_wfmt_row_bytes(fmt, K)


def repack_row_q6_K(src, K):
    """Host repack of one GGUF Q6_K row (bytes) to the SoA layout (gemv.hip:1341-1350)."""
    import numpy as np
    src = np.ascontiguousarray(src, dtype=np.uint8)
    dst = np.empty_like(src)
    check(_lib.lib().qmm_repack_row_q6_K(src.ctypes.data, dst.ctypes.data, K), "repack_row_q6_K")
    return dst


def _repack(name, src, K, dst_bytes):
    import numpy as np
    src = np.ascontiguousarray(src, dtype=np.uint8)
    dst = np.empty(dst_bytes, dtype=np.uint8)
    check(getattr(_lib.lib(), "qmm_" + name)(src.ctypes.data, dst.ctypes.data, K), name)
    return dst


def repack_row_q8_0(src, K):
    """Host repack of one GGUF Q8_0 row to the Q8_0_SOA layout (gemv.h:16, gemv.hip:1351-1354)."""
    return _repack("repack_row_q8_0", src, K, K + K // 16)


def repack_row_q5_1(src, K):
    """Host repack of one GGUF Q5_1 row to the Q5_1_SOA layout (gemv.h:17, gemv.hip:1458-1465)."""
    return _repack("repack_row_q5_1", src, K, K // 32 * 24)


def repack_row_q5_0(src, K):
    """Host repack of one GGUF Q5_0 row to the Q5_1_SOA layout, m = -16 d (gemv.h:18, gemv.hip:1448-1457)."""
    return _repack("repack_row_q5_0", src, K, K // 32 * 24)


def repack_interleave8(fmt, src, N, K):
    """Host 8-row block interleave of a whole matrix (gemv.h:21, gemv.hip:1442-1447)."""
    import numpy as np
    src = np.ascontiguousarray(src, dtype=np.uint8)
    dst = np.empty_like(src)
    check(_lib.lib().qmm_repack_interleave8(fmt, src.ctypes.data, dst.ctypes.data, N, K), "repack_interleave8")
    return dst


def wmma_il_bytes(fmt, N, K):
    return _lib.lib().qmm_wmma_il_bytes(fmt, N, K)


def repack_wmma_il(fmt, src, N, K):
    """Host 16-row piece-major layout of a whole matrix (gemv.h:37-38, gemv.hip:1280-1303)."""
    import numpy as np
    src = np.ascontiguousarray(src, dtype=np.uint8)
    dst = np.empty(wmma_il_bytes(fmt, N, K), dtype=np.uint8)
    check(_lib.lib().qmm_repack_wmma_il(fmt, src.ctypes.data, dst.ctypes.data, N, K), "repack_wmma_il")
    return dst


def quantize_x_q8(x, out, ncol, K, stream=None):
    """gemv.h:10: x f32 [ncol][K] -> out (XQ8Buf)."""
    _dev(x, torch.float32, "x")
    check(_lib.lib().qmm_quantize_x_q8(_p(x), out.c(), ncol, K, _stream(stream)), "quantize_x_q8")


def gemv_q8(fmt, W, x, y, N, K, ncol, tpr=0, rpt=1, stream=None):
    """gemv.h:25: y[c][n] = W[n] . x[c] for c < ncol (x an XQ8Buf)."""
    _dev(W, torch.uint8, "W"); _dev(y, torch.float32, "y")
    check(_lib.lib().qmm_gemv_q8(fmt, _p(W), x.c(), _p(y), N, K, ncol, tpr, rpt, _stream(stream)), "gemv_q8")


def _segs(segs):
    arr = (GemvSeg * len(segs))()
    for i, (fmt, w, y, N, K) in enumerate(segs):
        arr[i] = GemvSeg(fmt, w.data_ptr(), y.data_ptr(), N, K)
    return arr


def gemv_multi(segs, x, ncol, stream=None):
    """gemv.h:28: segs = [(fmt, W, y, N, K), ...] sharing x."""
    arr = _segs(segs)
    check(_lib.lib().qmm_gemv_multi(arr, len(segs), x.c(), ncol, _stream(stream)), "gemv_multi")


def gemv_wmma_ok(segs):
    """gemv.h:35: the library's GEMV is T-invariant for every supported format, so any segment list
    of Q4_K / Q6_K_SOA weights with K % 256 == 0 qualifies."""
    return 1 <= len(segs) <= 4 and all(f in (WFmt.Q4_K, WFmt.Q6_K_SOA) and K % 256 == 0 for f, _, _, _, K in segs)


def gemv_wmma(segs, x, ncol, mode=0, stream=None):
    """gemv.h:36: the reference's T-invariant matrix-core GEMV; here the (T-invariant) multi GEMV,
    mode accepted and ignored."""
    gemv_multi(segs, x, ncol, stream)


def gemv_splitk(fmt, W, x, part, N, K, ksplit, ncol, stream=None):
    """gemv.h:55: part[(c*ksplit + ks)][N] = W . x over the ks-th range of 256-weight blocks."""
    _dev(W, torch.uint8, "W"); _dev(part, torch.float32, "part")
    check(_lib.lib().qmm_gemv_splitk(fmt, _p(W), x.c(), _p(part), N, K, ksplit, ncol, _stream(stream)), "gemv_splitk")


def quantize_x_q8k(x, out, ncol, K, stream=None):
    """gemv.h:34: x f32 [ncol][K] -> out (XQ8KBuf): one scale per 256, int16 sums per 32."""
    _dev(x, torch.float32, "x")
    check(_lib.lib().qmm_quantize_x_q8k(_p(x), out.c(), ncol, K, _stream(stream)), "quantize_x_q8k")


def gemv_wmma_q8k(segs, x, ncol, ks_mode=0, stream=None):
    """gemv.h:35: segs = [(fmt, W, y, N, K), ...] on Q8_K activations (x an XQ8KBuf); ks_mode accepted."""
    arr = _segs(segs)
    check(_lib.lib().qmm_gemv_q8k(arr, len(segs), x.c(), ncol, _stream(stream)), "gemv_wmma_q8k")


def gemv_q8_f32x(fmt, W, x, y, N, K, ncol, stream=None):
    """quantize_x_q8 + gemv_q8 in one launch (f32 x in), bit for bit the same y."""
    check(_lib.lib().qmm_gemv_q8_f32x(fmt, _p(W), _p(x), _p(y), N, K, ncol, _stream(stream)), "gemv_q8_f32x")


def gemv_q4_K_f32(W, x, y, N, K, ncol, tpr=0, stream=None):
    """gemv.h:57: f32-activation Q4_K GEMV."""
    _dev(W, torch.uint8, "W"); _dev(x, torch.float32, "x"); _dev(y, torch.float32, "y")
    check(_lib.lib().qmm_gemv_q4_K_f32(_p(W), _p(x), _p(y), N, K, ncol, tpr, _stream(stream)), "gemv_q4_K_f32")


def moe_route(logits, ids, w, T, stream=None):
    """fn.h:43: logits [T][513] -> ids/w [T][11] (10 routed + shared)."""
    check(_lib.lib().qmm_moe_route(_p(logits), _p(ids), _p(w), T, _stream(stream)), "moe_route")


def moe_route_n(logits, ids, w, T, nexp, stride, topk, stream=None):
    check(_lib.lib().qmm_moe_route_n(_p(logits), _p(ids), _p(w), T, nexp, stride, topk, _stream(stream)), "moe_route_n")


def gemv_moe(fmt, shared_fmt, w, shared, y, ebytes, ids, nexp, x, N, K, T, xrow_te, slotw=None, stream=None):
    """gemv.h:44: w/shared/y are lists of 1 or 2 tensors (gate|up share a launch)."""
    nseg = len(w)
    a = MoeSegs()
    for g in range(nseg):
        a.w[g] = w[g].data_ptr(); a.shared[g] = shared[g].data_ptr(); a.y[g] = y[g].data_ptr()
    a.ebytes = ebytes
    a.slotw = 0 if slotw is None else slotw.data_ptr()
    check(_lib.lib().qmm_gemv_moe(fmt, shared_fmt, ctypes.byref(a), nseg, _p(ids), nexp, x.c(), N, K, T, int(xrow_te),
                                  _stream(stream)), "gemv_moe")


def moe_decode_ws_bytes(T, topk, F):
    return _lib.lib().qmm_moe_decode_ws_bytes(T, topk, F)


def moe_decode(fmt, Wg, Wu, Wd, ebytes_gu, ebytes_d, Sg, Su, Sd, logits, stride, nexp_total, topk, x, T, H, F, ids, w, ws, y,
               stream=None):
    """The MoE decode step in one call (T = 1: two launches, routing + gate|up + silu * up -> q8, then the
    down projection; T > 1: the four launches); ids / w [T][topk+1] and y [T][H] out, bitwise moe_route + gemv_moe +
    moe_silu_quant + gemv_moe.  ws: a device buffer of moe_decode_ws_bytes(T, topk, F) bytes."""
    check(_lib.lib().qmm_moe_decode(fmt, _p(Wg), _p(Wu), _p(Wd), ebytes_gu, ebytes_d, _p(Sg), _p(Su), _p(Sd), _p(logits), stride,
                                    nexp_total, topk, x.c(), T, H, F, _p(ids), _p(w), _p(ws), ws.numel() * ws.element_size(),
                                    _p(y), _stream(stream)), "moe_decode")


def moe_decode_noalloc(fmt, Wg, Wu, Wd, ebytes_gu, ebytes_d, Sg, Su, Sd, logits, stride, nexp_total, topk, x, T, H, F, ids, w, y,
                       stream=None):
    """moe_decode with its workspace in the library's static per-GPU array (no allocation; calls that
    overlap on one GPU race); QmmError(-5) when moe_decode_ws_bytes(T, topk, F) > moe_decode_scratch_max()."""
    check(_lib.lib().qmm_moe_decode_noalloc(fmt, _p(Wg), _p(Wu), _p(Wd), ebytes_gu, ebytes_d, _p(Sg), _p(Su), _p(Sd), _p(logits),
                                            stride, nexp_total, topk, x.c(), T, H, F, _p(ids), _p(w), _p(y), _stream(stream)),
          "moe_decode_noalloc")


def moe_decode_scratch_max():
    return _lib.lib().qmm_moe_decode_scratch_max()


def moe_combine_sorted(down, w, kpos, y, T, nexp, E, stream=None):
    """fn.h:38: y[t][d] = sum_e w[t*nexp+e] * down[kpos[t*nexp+e]][d] (E is an argument here)."""
    check(_lib.lib().qmm_moe_combine_sorted(_p(down), _p(w), _p(kpos), _p(y), T, nexp, E, _stream(stream)),
          "moe_combine_sorted")


def moe_silu_quant(gate, up, xq, rows, n, stream=None):
    """fn.h:48: h = silu(g)*u quantised per 32 into xq (XQ8Buf of rows x n)."""
    check(_lib.lib().qmm_moe_silu_quant(_p(gate), _p(up), xq.c(), rows, n, _stream(stream)), "moe_silu_quant")


def f32_gemv(W, x, y, N, K, T, stream=None):
    """fn.h:37: y[t][n] = W[n] . x[t] in f32 (the reference's arithmetic and order)."""
    _dev(W, torch.float32, "W"); _dev(x, torch.float32, "x"); _dev(y, torch.float32, "y")
    check(_lib.lib().qmm_f32_gemv(_p(W), _p(x), _p(y), N, K, T, _stream(stream)), "f32_gemv")


def gemm_f32(A, W, D, M, N, K, stream=None):
    """gemm.h:31 (BlasLt::gemm_f32, the prefill router): D[m][n] = A[m] . W[n] in f32 on the matrix cores."""
    _dev(A, torch.float32, "A"); _dev(W, torch.float32, "W"); _dev(D, torch.float32, "D")
    check(_lib.lib().qmm_gemm_f32(_p(A), _p(W), _p(D), M, N, K, _stream(stream)), "gemm_f32")


def moe_router(Wr, x, logits, ids, w, T, nexp=512, K=None, topk=10, stream=None):
    """qwen4exp.cpp:346-347 in one call: logits = Wr . x (f32_gemv), then moe_route_n on them."""
    _dev(Wr, torch.float32, "Wr"); _dev(x, torch.float32, "x"); _dev(logits, torch.float32, "logits")
    K = x.shape[-1] if K is None else K
    check(_lib.lib().qmm_moe_router(_p(Wr), _p(x), _p(logits), _p(ids), _p(w), T, nexp, K, topk, _stream(stream)),
          "moe_router")


# ---- activation producers (engine/kernels/ops.h) ----
def add_rmsnorm_quant(x, y, w, xn, xq, T, n, eps, stream=None):
    """ops.h:14: per row, x += y (y may be None), xn = rmsnorm(x) * w, xq = q8(xn) (XQ8Buf of T x n)."""
    _dev(x, torch.float32, "x"); _dev(w, torch.float32, "w"); _dev(xn, torch.float32, "xn")
    if y is not None:
        _dev(y, torch.float32, "y")
    check(_lib.lib().qmm_add_rmsnorm_quant(_p(x), 0 if y is None else _p(y), _p(w), _p(xn), xq.c(), T, n, eps,
                                           _stream(stream)), "add_rmsnorm_quant")


def add_rmsnorm_bf16(x, y, w, xb, T, n, eps, stream=None):
    """ops.h:18: per row, x += y (y may be None), xb = bf16(rmsnorm(x) * w) (xb int16/uint16/bfloat16 storage)."""
    _dev(x, torch.float32, "x"); _dev(w, torch.float32, "w")
    if y is not None:
        _dev(y, torch.float32, "y")
    check(_lib.lib().qmm_add_rmsnorm_bf16(_p(x), 0 if y is None else _p(y), _p(w), _p(xb), T, n, eps,
                                          _stream(stream)), "add_rmsnorm_bf16")


def silu_mul_quant(gate, up, xq, n, stream=None):
    """ops.h:24: xq = q8(silu(gate) * up) per 32 over n values."""
    _dev(gate, torch.float32, "gate"); _dev(up, torch.float32, "up")
    check(_lib.lib().qmm_silu_mul_quant(_p(gate), _p(up), xq.c(), n, _stream(stream)), "silu_mul_quant")


def silu_mul_bf16(gate, up, out, n, stream=None):
    """ops.h:20: out = bf16(silu(gate) * up) over n values."""
    _dev(gate, torch.float32, "gate"); _dev(up, torch.float32, "up")
    check(_lib.lib().qmm_silu_mul_bf16(_p(gate), _p(up), _p(out), n, _stream(stream)), "silu_mul_bf16")


# ---- prefill GEMM (engine/kernels/gemm.h) ----
def dequant_bf16(fmt, W, out, N, K, stream=None):
    """gemm.h:12: W -> bf16 [N][K] (out: int16/uint16-sized tensor of N*K elements), bit-exact."""
    _dev(W, torch.uint8, "W")
    check(_lib.lib().qmm_dequant_bf16(fmt, _p(W), _p(out), N, K, _stream(stream)), "dequant_bf16")


def gemm_wq(fmt, W, A, D, M, N, K, stream=None):
    """D[M][N] f32 = A[M][K] bf16 . dequant(W)[N][K]^T, dequantisation fused into the GEMM."""
    _dev(W, torch.uint8, "W"); _dev(A, torch.bfloat16, "A"); _dev(D, torch.float32, "D")
    check(_lib.lib().qmm_gemm_wq(fmt, _p(W), _p(A), _p(D), M, N, K, _stream(stream)), "gemm_wq")


def gemm_bf16(A, W, D, M, N, K, stream=None):
    """BlasLt::gemm (gemm.h:27): D[M][N] bf16 = A[M][K] bf16 . W[N][K]^T bf16, f32 accumulate."""
    _dev(A, torch.bfloat16, "A"); _dev(W, torch.bfloat16, "W"); _dev(D, torch.bfloat16, "D")
    check(_lib.lib().qmm_gemm_bf16(_p(A), _p(W), _p(D), M, N, K, _stream(stream)), "gemm_bf16")


def gemm_bf16_ld(A, lda, W, ldw, D, M, N, K, stream=None):
    """BlasLt::gemm_ld (gemm.h:29): as gemm_bf16 with row strides lda / ldw (elements); A and W may be views."""
    check(_lib.lib().qmm_gemm_bf16_ld(_p(A), lda, _p(W), ldw, _p(D), M, N, K, _stream(stream)), "gemm_bf16_ld")


def gemm_tile(fmt, M, N, K):
    """Index of the tile that gemm_wq (fmt < 0: gemm_bf16) runs for this shape."""
    return _lib.lib().qmm_gemm_tile(fmt, M, N, K)


def f32_to_bf16(x, out, n, stream=None):
    check(_lib.lib().qmm_f32_to_bf16(_p(x), _p(out), n, _stream(stream)), "f32_to_bf16")


def bf16_to_f32(x, out, n, stream=None):
    check(_lib.lib().qmm_bf16_to_f32(_p(x), _p(out), n, _stream(stream)), "bf16_to_f32")


def bf16_to_f32_seg(x, Nt, off, N, out, M, stream=None):
    check(_lib.lib().qmm_bf16_to_f32_seg(_p(x), Nt, off, N, _p(out), M, _stream(stream)), "bf16_to_f32_seg")


def bf16_to_f32_seg2(x, x2, Nt, off, N, out, M, stream=None):
    check(_lib.lib().qmm_bf16_to_f32_seg2(_p(x), _p(x2), Nt, off, N, _p(out), M, _stream(stream)), "bf16_to_f32_seg2")


# ---- MoE prefill ----
MOE_TILE_ROWS = 128    # rows per tile of qmm_moe_gemm_bf16 / qmm_moe_gemm_gate_up_bf16 (at most 128)


def moe_tiles_capacity(T, nslot, nexperts, maxc=MOE_TILE_ROWS):
    return -(-(T * nslot) // maxc) + nexperts + 1


def moe_sort(ids, T, nslot, nexperts, maxc, kpos, rowtok, tiles, counts, stream=None):
    """Device expert sort (replaces the host path of qwen4exp.cpp:628-645).  tiles: int32 [cap][3]."""
    check(_lib.lib().qmm_moe_sort(_p(ids), T, nslot, nexperts, maxc, _p(kpos), _p(rowtok), _p(tiles), _p(counts),
                                  _stream(stream)), "moe_sort")


def moe_gemm_bf16(fmt, shared_fmt, W, Wsh, ebytes, tiles, counts, max_tiles, rowtab, A, D, N, K, stream=None):
    """Grouped expert GEMM over sorted rows, bf16 activations (moe_gemm, gemv.h:49-50)."""
    check(_lib.lib().qmm_moe_gemm_bf16(fmt, shared_fmt, _p(W), _p(Wsh), ebytes, _p(tiles), _p(counts), max_tiles,
                                       _p(rowtab), _p(A), _p(D), N, K, _stream(stream)), "moe_gemm_bf16")


def moe_gemm_gate_up_bf16(fmt, shared_fmt, Wg, Wgsh, Wu, Wush, ebytes, tiles, counts, max_tiles, rowtab, A, H, N, K,
                          stream=None):
    """h = bf16(silu(A . Wg^T) * (A . Wu^T)) over the sorted rows, one launch (gate, up and silu)."""
    check(_lib.lib().qmm_moe_gemm_gate_up_bf16(fmt, shared_fmt, _p(Wg), _p(Wgsh), _p(Wu), _p(Wush), ebytes, _p(tiles),
                                               _p(counts), max_tiles, _p(rowtab), _p(A), _p(H), N, K, _stream(stream)),
          "moe_gemm_gate_up_bf16")


def moe_silu_bf16(gate, up, h, n, stream=None):
    check(_lib.lib().qmm_moe_silu_bf16(_p(gate), _p(up), _p(h), n, _stream(stream)), "moe_silu_bf16")


def moe_gemm(fmt, shared_fmt, W, Wsh, ebytes, tiles, ntiles, stiles, nstiles, ct, rowtab, x, y, N, K, stream=None):
    """moe_gemm (gemv.h:49-50) with the reference's signature: q8 activations (x an XQ8Buf), routed tiles
    tiles[:ntiles] and shared tiles stiles[:nstiles] with host counts; y[k][N] f32, the q8 arithmetic."""
    check(_lib.lib().qmm_moe_gemm_q8(fmt, shared_fmt, _p(W), _p(Wsh), ebytes, _p(tiles), ntiles, _p(stiles), nstiles, ct,
                                     _p(rowtab), x.c(), _p(y), N, K, _stream(stream)), "moe_gemm")


# ---- MXFP4 decoder blocks ----
# These calls answer in a few microseconds on the device, so their checks are kept to one pass over each
# tensor and the arguments go to the library as plain integers.
_INT_MAX = (1 << 31) - 1
_DTYPE = {torch.float32: _lib.QMM_F32, torch.bfloat16: _lib.QMM_BF16}
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda d: torch.cuda.current_stream(d).cuda_stream)


def _handle(stream):
    """The stream to launch on: the current one of the current device, or one of that device."""
    if stream is None:
        return _raw_stream(_device())
    if stream.device_index != _device():
        raise QmmError(f"the stream is of cuda:{stream.device_index}, the current device is cuda:{_device()}")
    return stream.cuda_stream


def _in(t, n, name, dtype=None):
    """The address of t: a contiguous tensor of at least n elements on the current device (the library launches there)."""
    if t is None or not t.is_cuda or (dtype is not None and t.dtype is not dtype) or not t.is_contiguous():
        _dev(t, dtype, name)
    if t.get_device() != _device():
        raise QmmError(f"{name} is on {t.device}, the current device is cuda:{_device()}")
    if t.numel() < n:
        raise QmmError(f"{name} holds {t.numel()} elements, {n} are needed")
    return t.data_ptr()


def _dtype(t, name):
    d = _DTYPE.get(t.dtype)
    if d is None:
        raise QmmError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    return d


def _rows(t, rows, n, name):
    """The row stride of t, `rows` rows of n contiguous values (or one row [n]) on the current device."""
    if t is None or not t.is_cuda:
        raise QmmError(f"{name} must be a CUDA tensor")
    if t.get_device() != _device():
        raise QmmError(f"{name} is on {t.device}, the current device is cuda:{_device()}")
    shape = t.shape
    if len(shape) not in (1, 2) or shape[-1] != n or (n > 1 and t.stride(-1) != 1):
        raise QmmError(f"{name} must be rows of {n} contiguous values, got shape {tuple(shape)}, strides {tuple(t.stride())}")
    have = shape[0] if len(shape) == 2 else 1
    if have < rows:
        raise QmmError(f"{name} has {have} rows, {rows} are needed")
    if have == 1:
        return n
    ld = t.stride(0)
    if ld < n:
        raise QmmError(f"{name}: rows overlap (stride {ld}, {n} values)")
    return ld


def mxfp4_steps(K):
    """Steps of 128 values that a row of K takes."""
    return -(-K // 128)


class XMXBuf:
    """Device buffers of rows of MXFP4: q [rows][64 per step of 128] uint8, e [rows][4 per step] uint8."""

    def __init__(self, rows, K, device="cuda"):
        self.rows, self.K = rows, K
        self.q = torch.zeros((rows, 64 * mxfp4_steps(K)), dtype=torch.uint8, device=device)
        self.e = torch.zeros((rows, 4 * mxfp4_steps(K)), dtype=torch.uint8, device=device)

    def c(self):
        return XMX(self.q.data_ptr(), self.e.data_ptr())


def _xmx(x, rows, K, name):
    steps = (K + 127) // 128
    if (x.K + 127) // 128 != steps:
        raise QmmError(f"{name} holds rows of {x.K} values, rows of {K} are needed")
    return XMX(_in(x.q, rows * steps * 64, name, torch.uint8), _in(x.e, rows * steps * 4, name, torch.uint8))


def quantize_mxfp4(x, out, rows, K, stream=None):
    """x f32 or bf16 [rows][K] (rows may be strided) -> out (XMXBuf): blocks of 32, scale 2^(floor(log2 amax) - 2),
    codes rounded to nearest even."""
    ld = _rows(x, rows, K, "x")
    check(_lib.lib().qmm_quantize_mxfp4(x.data_ptr(), _dtype(x, "x"), ld, _xmx(out, rows, K, "out"), rows, K, _handle(stream)), "quantize_mxfp4")


def dequant_mxfp4(x, out, rows, K, stream=None):
    """The values of x (XMXBuf) into out [rows][K], f32 or bf16 (exact in both)."""
    check(_lib.lib().qmm_dequant_mxfp4(_xmx(x, rows, K, "x"), _in(out, rows * K, "out"), _dtype(out, "out"), rows, K, _handle(stream)), "dequant_mxfp4")


def mxfp4_weight_bytes(N, K):
    """Bytes of a packed MXFP4 weight of N rows of K values."""
    return _lib.lib().qmm_mxfp4_weight_bytes(N, K)


def _wbytes(N, K):
    steps = (K + 127) // 128
    return (N + 15) // 16 * (steps * 1024 + (steps + 3) // 4 * 256)


def _weight(W, N, K, name="W", extra=0):
    """The address of a packed weight of N rows of K values, `extra` bytes into its buffer."""
    return _in(W, extra + _wbytes(N, K), name, torch.uint8)


def _experts(W, N, K, ebytes, n):
    """The address of n packed weights of N rows of K values, `ebytes` apart."""
    if ebytes < 0:
        raise QmmError(f"W: weights {ebytes} bytes apart")
    return _weight(W, N, K, "W", (n - 1) * ebytes)


def pack_mxfp4(q, e, W, N, K, stream=None):
    """MXFP4 rows q [N][64 per step], e [N][4 per step] (an XMXBuf's tensors) -> W, the layout the products read."""
    for t, per, name in ((q, 64, "q"), (e, 4, "e")):
        _in(t, 0, name, torch.uint8)
        if t.numel() != N * per * mxfp4_steps(K):
            raise QmmError(f"{name} must hold {N} rows of {per * mxfp4_steps(K)} bytes")
    check(_lib.lib().qmm_pack_mxfp4(XMX(q.data_ptr(), e.data_ptr()), _weight(W, N, K), N, K, _handle(stream)), "pack_mxfp4")


def repack_row_mxfp4(src, K):
    """Host: one GGUF row of MXFP4 blocks (bytes) -> (q, e) bytes of one MXFP4 row."""
    import numpy as np
    src = np.ascontiguousarray(src, dtype=np.uint8)
    if K > 0 and src.size != K // 32 * 17:
        raise QmmError(f"a GGUF MXFP4 row of {K} weights has {K // 32 * 17} bytes, got {src.size}")
    q, e = np.empty(64 * mxfp4_steps(K), np.uint8), np.empty(4 * mxfp4_steps(K), np.uint8)
    check(_lib.lib().qmm_repack_row_mxfp4(src.ctypes.data, q.ctypes.data, e.ctypes.data, K), "repack_row_mxfp4")
    return q, e


def gemv_mxfp4(W, x, y, ncol, N, K, stream=None):
    """y[m][n] = W[n] . x[m] for m < ncol <= 64 (x an XMXBuf, y f32 or bf16 [ncol][N])."""
    check(_lib.lib().qmm_gemv_mxfp4(_weight(W, N, K), _xmx(x, ncol, K, "x"), _in(y, ncol * N, "y"), _dtype(y, "y"), ncol, N, K, _handle(stream)),
          "gemv_mxfp4")


def gemm_mxfp4(W, x, D, M, N, K, stream=None):
    """D[m][n] = W[n] . x[m] for any M (x an XMXBuf, D f32 or bf16 [M][N])."""
    check(_lib.lib().qmm_gemm_mxfp4(_weight(W, N, K), _xmx(x, M, K, "x"), _in(D, M * N, "D"), _dtype(D, "D"), M, N, K, _handle(stream)), "gemm_mxfp4")


def gemm_mxfp4_tile(M, N, K):
    """Index of the tile that gemm_mxfp4 runs for this shape."""
    return _lib.lib().qmm_gemm_mxfp4_tile(M, N, K)


def gemv_moe_mxfp4(W, Wsh, ebytes, ids, x, y, T, nslot, nexperts, N, K, xrow_te=False, stream=None):
    """y[te][n] = W_{ids[te]}[n] . x[te if xrow_te else t] for T <= 16 tokens (ids int32 [T][nslot], below 0: Wsh)."""
    slots = T * nslot
    check(_lib.lib().qmm_gemv_moe_mxfp4(_experts(W, N, K, ebytes, nexperts), None if Wsh is None else _weight(Wsh, N, K, "Wsh"), ebytes,
                                        _in(ids, slots, "ids", torch.int32), _xmx(x, slots if xrow_te else T, K, "x"), _in(y, slots * N, "y"),
                                        _dtype(y, "y"), T, nslot, nexperts, N, K, int(xrow_te), _handle(stream)), "gemv_moe_mxfp4")


def moe_gemm_mxfp4(W, Wsh, ebytes, tiles, counts, max_tiles, rowtab, x, D, N, K, stream=None, rows=None, nexperts=None):
    """D[k] = W_e . x[rowtab[k]] over rows sorted by expert (moe_sort's tiles, counts, rowtok; rowtab None: x[k]).

    rows: how many the tiles hold at most, which D and rowtab must have room for (None: as many as rowtab has, or without
    it x); nexperts: of W (None: as many as it holds).  Tiles that name others reach nothing outside the tensors."""
    pw = _experts(W, N, K, ebytes, 1 if nexperts is None else nexperts)
    if nexperts is None:
        nexperts = min(1 + (W.numel() - _wbytes(N, K)) // ebytes, _INT_MAX) if ebytes else 1
    xrows = min(x.q.numel() // (64 * max(1, (K + 127) // 128)), _INT_MAX)
    if rows is None:
        rows = xrows if rowtab is None else rowtab.numel()
    check(_lib.lib().qmm_moe_gemm_mxfp4_n(pw, None if Wsh is None else _weight(Wsh, N, K, "Wsh"), ebytes, nexperts,
                                          _in(tiles, 3 * max_tiles, "tiles", torch.int32), _in(counts, 2, "counts", torch.int32), max_tiles,
                                          None if rowtab is None else _in(rowtab, rows, "rowtab", torch.int32), rows, _xmx(x, xrows, K, "x"), xrows,
                                          _in(D, rows * N, "D"), _dtype(D, "D"), N, K, _handle(stream)), "moe_gemm_mxfp4")


_SCORE = {"softmax": 0, "sigmoid": 1}
_SHARED = {None: 0, "gate": 1, "one": 2}


def moe_route_groups(logits, ids, w, T, nexp, topk, score="softmax", bias=None, groups=1, keep=1, best=1, renorm=True, scale=1.0, shared=None,
                     stream=None):
    """Experts of each token: scores (softmax or sigmoid of logits [T][>= nexp]), plus bias for the choice, the `keep`
    best of `groups` groups (by their `best` = 1 or 2 largest), the topk experts of those (ties to the lower id);
    weights: the scores, renormalised if renorm, times scale.  shared: None, "gate" (logit nexp's sigmoid) or "one",
    a last slot of id -1.  ids int32, w f32 [T][topk (+ 1)]."""
    if score not in _SCORE or shared not in _SHARED:
        raise QmmError(f"score {score!r}, shared {shared!r}: softmax or sigmoid; None, 'gate' or 'one'")
    stride, slots = logits.shape[-1], T * (topk + (shared is not None))
    rule = RouteRule(None if bias is None else _in(bias, nexp, "bias", torch.float32), scale, _SCORE[score], groups, keep, best, int(renorm),
                     _SHARED[shared])
    check(_lib.lib().qmm_moe_route_groups(_in(logits, T * stride, "logits", torch.float32), stride, rule, _in(ids, slots, "ids", torch.int32),
                                          _in(w, slots, "w", torch.float32), T, nexp, topk, _handle(stream)), "moe_route_groups")


_ACT = {"none": 0, "sigmoid": 1, "silu": 2}


def _postnorm(x, y, wy, w, gate, act, alpha, xo, T, n):
    """The leading arguments of the postnorm_add_rmsnorm calls."""
    px = _in(x, T * n, "x", torch.float32)
    ldy = _rows(y, T, n, "y")
    if act not in _ACT:
        raise QmmError(f"act {act!r}: none, sigmoid or silu")
    g = None
    if gate is not None:
        if gate.dim() == 2 and gate.shape[1] == 1 and n > 1:             # one value per token
            _rows(gate, T, 1, "gate")
            ld, per = gate.stride(0), 0
        elif gate.dim() == 1:                                            # one row for every token
            _rows(gate, 1, n, "gate")
            ld, per = 0, 1
        else:
            ld, per = _rows(gate, T, n, "gate"), 1
        g = Gate(gate.data_ptr(), ld, _dtype(gate, "gate"), _ACT[act], per)
    return (px, y.data_ptr(), _dtype(y, "y"), ldy, None if wy is None else _in(wy, n, "wy", torch.float32), g, alpha,
            px if xo is None else _in(xo, T * n, "xo", torch.float32), _in(w, n, "w", torch.float32))


def postnorm_add_rmsnorm_bf16(x, y, wy, w, xb, T, n, eps, gate=None, act="none", alpha=1.0, xo=None, stream=None):
    """Between two blocks, per row: p = rmsnorm(y) * wy (wy None: y), p *= act(gate), xo = x + alpha * p (xo None: in
    place), xb = bf16(rmsnorm(xo) * w).  y f32 or bf16 rows; gate f32 or bf16 [T][1], [n] or [T][n]."""
    a = _postnorm(x, y, wy, w, gate, act, alpha, xo, T, n)
    check(_lib.lib().qmm_postnorm_add_rmsnorm_bf16(*a, _in(xb, T * n, "xb", torch.bfloat16), T, n, eps, _handle(stream)), "postnorm_add_rmsnorm_bf16")


def postnorm_add_rmsnorm_quant(x, y, wy, w, xn, xq, T, n, eps, gate=None, act="none", alpha=1.0, xo=None, stream=None):
    """The same with xn = rmsnorm(xo) * w in f32 and its q8 in xq (XQ8Buf of T x n); n % 32 == 0."""
    a = _postnorm(x, y, wy, w, gate, act, alpha, xo, T, n)
    if xq.ncol < T or xq.K != n:
        raise QmmError(f"xq holds {xq.ncol} rows of {xq.K} values, {T} of {n} are needed")
    dev = _device()
    if xq.q.get_device() != dev or xq.d.get_device() != dev or xq.s.get_device() != dev or (xq.ds is not None and xq.ds.get_device() != dev):
        raise QmmError(f"xq is on {xq.q.device}, the current device is cuda:{dev}")
    check(_lib.lib().qmm_postnorm_add_rmsnorm_quant(*a, _in(xn, T * n, "xn", torch.float32), xq.c(), T, n, eps, _handle(stream)),
          "postnorm_add_rmsnorm_quant")


def postnorm_add_rmsnorm_mxfp4(x, y, wy, w, xq, T, n, eps, gate=None, act="none", alpha=1.0, xo=None, stream=None):
    """The same with rmsnorm(xo) * w as MXFP4 rows (XMXBuf of T x n)."""
    a = _postnorm(x, y, wy, w, gate, act, alpha, xo, T, n)
    check(_lib.lib().qmm_postnorm_add_rmsnorm_mxfp4(*a, _xmx(xq, T, n, "xq"), T, n, eps, _handle(stream)), "postnorm_add_rmsnorm_mxfp4")


# ---- attention between a block's q, k, v products and its output product ----
class KVMXBuf:
    """A cache of keys and values in MXFP4, in pages of `page` tokens: kq, vq [pages][heads][page][dim / 2] uint8 (codes), ke, ve
    [pages][heads][page][dim / 32] uint8 (scale bytes)."""

    def __init__(self, pages, page, heads, dim, device="cuda"):
        self.held = None                                 # what the calls checked, until a tensor or a size is set
        self.pages, self.page, self.heads, self.dim = pages, page, heads, dim
        self.kq, self.vq = (torch.zeros((pages, heads, page, dim // 2), dtype=torch.uint8, device=device) for _ in range(2))
        self.ke, self.ve = (torch.zeros((pages, heads, page, dim // 32), dtype=torch.uint8, device=device) for _ in range(2))

    def __setattr__(self, name, value):
        if name != "held":
            object.__setattr__(self, "held", None)
        object.__setattr__(self, name, value)

    def __getstate__(self):                              # copies check anew
        return {**self.__dict__, "held": None}

    def c(self):
        return KVMX(self.kq.data_ptr(), self.ke.data_ptr(), self.vq.data_ptr(), self.ve.data_ptr(), self.pages, self.page, self.heads, self.dim)


def _at(t, n, dtype, dev, name):
    """_in for calls that take many tensors: the address of t, contiguous, of this type, on the current device dev, n elements at least."""
    if t.dtype is dtype and t.get_device() == dev and t.is_contiguous() and t.numel() >= n:
        return t.data_ptr()
    return _in(t, n, name, dtype)


def _kv(kv, dev):
    """The cache as the library takes it, made anew when one of its tensors or sizes was set, has moved, was turned in place or has another
    number of elements, or the current device is another."""
    kq, ke, vq, ve, held = kv.kq, kv.ke, kv.vq, kv.ve, kv.held
    if (held is not None and held[1] == (kq.data_ptr(), ke.data_ptr(), vq.data_ptr(), ve.data_ptr(), kq.numel(), ke.numel(), vq.numel(), ve.numel(), dev)
            and kq.is_contiguous() and ke.is_contiguous() and vq.is_contiguous() and ve.is_contiguous()):
        return held[0]
    tokens, u8 = kv.pages * kv.heads * kv.page, torch.uint8
    q, e = tokens * (kv.dim // 2), tokens * (kv.dim // 32)
    p = (_at(kq, q, u8, dev, "kv.kq"), _at(ke, e, u8, dev, "kv.ke"), _at(vq, q, u8, dev, "kv.vq"), _at(ve, e, u8, dev, "kv.ve"))
    c = KVMX(*p, kv.pages, kv.page, kv.heads, kv.dim)
    kv.held = (c, (*p, kq.numel(), ke.numel(), vq.numel(), ve.numel(), dev))
    return c


def _seqs(cu, lens, table, dev):
    n, i32 = lens.numel(), torch.int32
    shape = table.shape
    if len(shape) != 2 or shape[0] < n:
        raise QmmError(f"table must have a row of pages for each of {n} sequences, got shape {tuple(shape)}")
    return Seqs(_at(cu, n + 1, i32, dev, "cu"), _at(lens, n, i32, dev, "lens"), _at(table, 0, i32, dev, "table"), n, shape[1])


def _heads(t, rows, heads, dim, dev, name):
    """The row stride of t, `rows` rows of heads * dim contiguous values: [rows][heads * dim] or [rows][heads][dim], or one such row."""
    n = heads * dim
    if t is not None and t.get_device() == dev:
        shape = t.shape
        if len(shape) == 2 and shape[0] >= rows and shape[1] == n and (n == 1 or t.stride(1) == 1):
            ld = t.stride(0) if shape[0] > 1 else n
            if ld >= n:
                return ld
        elif len(shape) == 3:
            if shape[1] != heads or shape[2] != dim or (dim > 1 and t.stride(2) != 1) or (heads > 1 and t.stride(1) != dim):
                raise QmmError(f"{name} must be rows of {heads} heads of {dim} contiguous values, got shape {tuple(shape)}, strides {tuple(t.stride())}")
            if shape[0] < rows:
                raise QmmError(f"{name} has {shape[0]} rows, {rows} are needed")
            ld = t.stride(0) if shape[0] > 1 else n
            if ld < n:
                raise QmmError(f"{name}: rows overlap (stride {ld}, {n} values)")
            return ld
    return _rows(t, rows, n, name)


_STYLE = {"halves": 0, "neighbours": 1}


def rope_axes(x, out, pos, freq, axis, rows, heads, dim, style="halves", scale=1.0, stream=None):
    """Rotary positions with several axes: pair i of every head of row t of x turns by pos[axis[i]][t] * freq[i], times scale.

    x, out: rows of heads * dim values, f32 or bf16 each (out may be x); pos int32 [axes][rows] or [rows]; freq f32 [pairs]; axis uint8
    [pairs] or None (axis 0 for all); style "halves" (values i and i + pairs are a pair) or "neighbours" (2 i and 2 i + 1).  Values
    from 2 pairs on are copied."""
    if style not in _STYLE:
        raise QmmError(f"style {style!r}: halves or neighbours")
    pairs = freq.numel()
    axes, ldp = (1, 0) if pos.dim() == 1 else (pos.shape[0], pos.shape[-1])
    if pos.dim() > 2 or (pos.shape[-1] < rows):
        raise QmmError(f"pos must be [axes][rows] or [rows] with {rows} rows, got shape {tuple(pos.shape)}")
    dev = _device()
    ldx, ldo = _heads(x, rows, heads, dim, dev, "x"), _heads(out, rows, heads, dim, dev, "out")
    r = Rope(_at(freq, pairs, torch.float32, dev, "freq"), None if axis is None else _at(axis, pairs, torch.uint8, dev, "axis"),
             _at(pos, 0, torch.int32, dev, "pos"), ldp, axes, pairs, _STYLE[style], scale)
    check(_lib.lib().qmm_rope_axes(x.data_ptr(), _dtype(x, "x"), ldx, out.data_ptr(), _dtype(out, "out"), ldo, r, rows, heads, dim, _handle(stream)),
          "rope_axes")


def _same(k, v, what):
    if k.dtype is not v.dtype:
        raise QmmError(f"{what} must be of one type, got {k.dtype} and {v.dtype}")
    return _dtype(k, "k")


def kv_write_mxfp4(k, v, kv, cu, lens, table, rows, stream=None):
    """k, v (f32 or bf16, `rows` rows of the cache's heads * dim) -> their tokens' places in kv (KVMXBuf), as MXFP4.

    Rows cu[b] .. cu[b + 1] - 1 are the last ones of sequence b, which has lens[b] tokens with them; table[b] are its pages (int32,
    all on the device).  Rows from the last cu on, and tokens outside the table or the cache, are not written."""
    dev, heads, dim = _device(), kv.heads, kv.dim
    ldk, ldv = _heads(k, rows, heads, dim, dev, "k"), _heads(v, rows, heads, dim, dev, "v")
    check(_lib.lib().qmm_kv_write_mxfp4(k.data_ptr(), ldk, v.data_ptr(), ldv, _same(k, v, "k and v"), _kv(kv, dev), _seqs(cu, lens, table, dev), rows,
                                        _handle(stream)), "kv_write_mxfp4")


def kv_read_mxfp4(kv, cu, lens, table, k, v, rows, stream=None):
    """The values that kv holds for the tokens of these rows (as kv_write_mxfp4 places them) -> k, v, f32 or bf16 (exact in both)."""
    dev, heads, dim = _device(), kv.heads, kv.dim
    ldk, ldv = _heads(k, rows, heads, dim, dev, "k"), _heads(v, rows, heads, dim, dev, "v")
    check(_lib.lib().qmm_kv_read_mxfp4(_kv(kv, dev), _seqs(cu, lens, table, dev), k.data_ptr(), ldk, v.data_ptr(), ldv, _same(k, v, "k and v"), rows,
                                       _handle(stream)), "kv_read_mxfp4")


def attn_kv_ws_bytes(rows, heads, dim, max_len):
    """Bytes of attn_kv_mxfp4's workspace (0: it needs none): every row and head has room for up to 128 chunks of the keys up to max_len."""
    return _lib.lib().qmm_attn_kv_ws_bytes(rows, heads, dim, max_len)


def _attn(scale, dim, window, sinks, heads, dev):
    return Attn(None if sinks is None else _at(sinks, heads, torch.float32, dev, "sinks"), dim ** -0.5 if scale is None else scale, window)


def attn_kv_mxfp4(q, kv, cu, lens, table, out, rows, heads, max_rows, max_len, ws, scale=None, window=0, sinks=None, stream=None):
    """Attention of up to max_rows (<= 16) new rows a sequence over the cache kv, which holds their keys and values already.

    q, out: `rows` rows of heads * kv.dim values, f32 or bf16 each; heads / kv.heads (<= 16) successive heads share one of the cache;
    max_len: at least the longest of lens; ws: a uint8 tensor of attn_kv_ws_bytes(rows, heads, kv.dim, max_len) bytes (None where that
    is 0); scale None: dim ** -0.5; window: keys a row sees with its own (0: all); sinks f32 [heads]: a logit beside the keys'.  Where q and
    out are bf16, weights are rounded to bf16 as factors of their products with the values."""
    dev, dim = _device(), kv.dim
    ldq, ldo = _heads(q, rows, heads, dim, dev, "q"), _heads(out, rows, heads, dim, dev, "out")
    check(_lib.lib().qmm_attn_kv_mxfp4(q.data_ptr(), _dtype(q, "q"), ldq, _kv(kv, dev), _seqs(cu, lens, table, dev), _attn(scale, dim, window, sinks, heads, dev),
                                       out.data_ptr(), _dtype(out, "out"), ldo, rows, heads, max_rows, max_len,
                                       None if ws is None else _at(ws, 0, torch.uint8, dev, "ws"), 0 if ws is None else ws.numel(), _handle(stream)),
          "attn_kv_mxfp4")


def attn_prompt_ws_bytes(rows, krows, nseq, heads, dim):
    """Bytes of attn_prompt_bf16's workspace, enough for any window (0: it needs none)."""
    return _lib.lib().qmm_attn_prompt_ws_bytes(rows, krows, nseq, heads, dim)


def attn_prompt_bf16(q, k, v, cu_q, cu_k, out, heads, kv_heads, dim, scale=None, window=0, sinks=None, ws=None, stream=None):
    """Causal attention of packed sequences: rows cu_q[b] .. cu_q[b + 1] - 1 of q, the last ones of the tokens cu_k[b] .. cu_k[b + 1] - 1
    of k and v (cu_k None: cu_q).  q, out rows of heads * dim values, k, v of kv_heads * dim, all bf16 (row strides multiples of 8);
    scale, window and sinks as in attn_kv_mxfp4.  ws: a uint8 tensor of attn_prompt_ws_bytes(...) bytes; None: torch's allocator gives one
    where few rows see many keys (False: none, the keys stay in one part).  Weights are rounded to bf16 as factors of their products with v."""
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        if t.dtype is not torch.bfloat16:
            raise QmmError(f"{name} must be torch.bfloat16, got {t.dtype}")
    rows, krows, n = q.shape[0], k.shape[0], cu_q.numel() - 1
    dev, L = _device(), _lib.lib()
    ldq, ldo = _heads(q, rows, heads, dim, dev, "q"), _heads(out, rows, heads, dim, dev, "out")
    ldk, ldv = _heads(k, krows, kv_heads, dim, dev, "k"), _heads(v, krows, kv_heads, dim, dev, "v")
    handle = _handle(stream)
    if ws is None:
        size = L.qmm_attn_prompt_ws_bytes(rows, krows, n, heads, dim)
        if size:
            with torch.cuda.stream(stream):              # of that stream's memory: what this one still uses is not given away
                ws = torch.empty(size, dtype=torch.uint8, device=q.device)
    pw, size = (_at(ws, 0, torch.uint8, dev, "ws"), ws.numel()) if ws is not None and ws is not False else (None, 0)
    check(L.qmm_attn_prompt_bf16(q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, out.data_ptr(), ldo, _at(cu_q, n + 1, torch.int32, dev, "cu_q"),
                                 None if cu_k is None else _at(cu_k, n + 1, torch.int32, dev, "cu_k"), n, _attn(scale, dim, window, sinks, heads, dev),
                                 rows, krows, heads, kv_heads, dim, pw, size, handle), "attn_prompt_bf16")
