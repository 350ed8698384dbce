"""Host-side wrappers: layout, padding and tile choice around the HIP kernels.

Drop-in for the reference's nkilab/ops.py: same names, signatures, argument
meaning, output dtype (= input dtype) and errors.  Every op takes NumPy arrays
(float32, or ml_dtypes.bfloat16 when installed) or torch tensors.  NumPy in
gives NumPy out, synchronously, as in the reference; torch GPU tensors stay on
the GPU and the call is asynchronous on torch's current HIP stream.

Where the reference calls ``nki.simulate(kernel)(...)`` (ops.py:48-90), these
wrappers call the C ABI of libnkilab_hip.so (include/nkilab_hip.h).  There is
no CPU fallback: without the library or a GPU the ops raise.

The ``*_into`` functions are the GPU-tensor layer underneath: they write into
a caller-provided output, accept strided views and never copy weights, and are
what nkilab.model uses.
"""
from __future__ import annotations

import math
import struct
from dataclasses import dataclass
from functools import lru_cache
from itertools import chain

import numpy as np
import torch

from . import _lib
from ._tensors import current_device, dtype_code, from_device, ptr, stream_handle, to_device, workspace

# Reference tile sizes (nkilab/kernels/matmul.py:19-21, attention.py:24).  They
# define choose_blocks' grid and _pad_to's semantics; the HIP kernels handle
# ragged shapes themselves and never need host padding.
TK, TM, TN = 128, 128, 512
T = 128


def _pad_to(x: np.ndarray, rows: int, cols: int) -> np.ndarray:
    """Zero-pad a 2-D array at the end of both axes (ops.py:19-24)."""
    if x.shape == (rows, cols):
        return np.ascontiguousarray(x)
    out = np.zeros((rows, cols), dtype=x.dtype)
    out[: x.shape[0], : x.shape[1]] = x
    return out


def choose_blocks(m_tiles: int, n_tiles: int) -> tuple[int, int]:
    """Largest BM x BN accumulator block with BM*BN <= 8 that divides the tile grid;
    among equal-size blocks the one with the larger BN (ops.py:27-35)."""
    cands = [(bm, bn) for bm in (1, 2, 4) for bn in (1, 2, 4, 8)
             if bm * bn <= 8 and m_tiles % bm == 0 and n_tiles % bn == 0]
    return max(cands, key=lambda c: (c[0] * c[1], c[1]))


# ------------------------------------------------------------------ GEMM --

_MATMUL_VARIANTS = {"blocked": _lib.GEMM_BLOCKED, "naive": _lib.GEMM_NAIVE}


def _row_major(t: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """(tensor, leading dim) with unit column stride."""
    if t.dim() == 2:
        ld, cs = t.stride()
        if (cs == 1 or t.shape[1] == 1) and ld >= cols and t.shape[0] > 0:
            return t, ld
    t = t.contiguous()
    return t, max(cols, 1)


def _gemm(a: torch.Tensor, bmat: torch.Tensor, ldb: int, b_trans: bool, c: torch.Tensor,
          residual: torch.Tensor | None, variant: str) -> torch.Tensor:
    # The C ABI takes bare pointers and sizes: every shape is checked here, so
    # that a mismatch raises instead of reading or writing past a buffer.
    if a.dim() != 2 or bmat.dim() != 2 or c.dim() != 2:
        raise ValueError(f"gemm: 2-D operands expected, got {tuple(a.shape)}, {tuple(bmat.shape)}, {tuple(c.shape)}")
    M, K = a.shape
    Mc, N = c.shape
    if Mc != M:
        raise ValueError(f"gemm: output {tuple(c.shape)} does not have the {M} rows of a {tuple(a.shape)}")
    if bmat.shape != ((N, K) if b_trans else (K, N)):
        want_b = (N, K) if b_trans else (K, N)
        raise ValueError(f"gemm: b {tuple(bmat.shape)} does not match [{'N, K' if b_trans else 'K, N'}] = {want_b}")
    if residual is not None and residual.shape != (M, N):
        raise ValueError(f"gemm: residual {tuple(residual.shape)} does not match the output [{M}, {N}]")
    if a.dtype != bmat.dtype:
        raise TypeError(f"gemm: a and b must share a dtype, got {a.dtype} and {bmat.dtype}")
    a, lda = _row_major(a, K)
    ldc, cs = c.stride()
    if (cs != 1 and N > 1) or (M > 1 and ldc < N):
        raise ValueError("gemm: the output must be a row-major [M, N] tensor")
    if M <= 1:
        ldc = max(N, 1)
    ldr = 0
    if residual is not None:
        residual, ldr = _row_major(residual, N)
    if M == 0 or N == 0:
        return c
    if K == 0:
        c.copy_(residual if residual is not None else torch.zeros_like(c))
        return c
    pa, pb, pc, st = a.data_ptr(), bmat.data_ptr(), c.data_ptr(), stream_handle()
    pr = None if residual is None else residual.data_ptr()
    dt_in, dt_out, bt = dtype_code(a.dtype), dtype_code(c.dtype), int(b_trans)
    if _MATMUL_VARIANTS[variant] == _lib.GEMM_NAIVE:
        _lib.call("nkl_gemm", pa, pb, pc, pr, M, N, K, lda, ldb, ldc, ldr, bt, 1, 0, 0, 0, 0, dt_in, dt_out,
                  _lib.GEMM_NAIVE, st)
        return c
    # Most shapes need no workspace; the call says so before it launches anything.
    L = _lib.lib()
    rc = L.nkl_gemm_ws(pa, pb, pc, pr, None, 0, M, N, K, lda, ldb, ldc, ldr, bt, dt_in, dt_out, st)
    if rc == _lib.EWORKSPACE:
        nbytes = L.nkl_gemm_workspace_bytes(pa, pb, M, N, K, lda, ldb, bt, dt_in, dt_out)
        try:
            ws = workspace(nbytes, c.device)
        except torch.OutOfMemoryError:  # a workspace only makes the product faster: run it without one
            rc = L.nkl_gemm(pa, pb, pc, pr, M, N, K, lda, ldb, ldc, ldr, bt, 1, 0, 0, 0, 0, dt_in, dt_out,
                            _lib.GEMM_BLOCKED, st)
        else:
            rc = L.nkl_gemm_ws(pa, pb, pc, pr, ws.data_ptr(), nbytes, M, N, K, lda, ldb, ldc, ldr, bt, dt_in, dt_out,
                               st)
    if rc:
        _lib.check("nkl_gemm_ws", rc)
    return c


def gemm_into(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, residual: torch.Tensor | None = None,
              variant: str = "blocked") -> torch.Tensor:
    """c = a @ b (+ residual) on the GPU; a: [M, K], b: [K, N], c: [M, N].
    A b stored column-major (e.g. ``w.t()`` of a row-major [N, K] weight) is
    read in place by the B^T kernel; no transpose copy is made."""
    K, N = b.shape
    s0, s1 = b.stride()
    if s0 == 1 and N > 1 and K > 1 and s1 >= K:
        return _gemm(a, b.t(), s1, True, c, residual, variant)
    bm, ldb = _row_major(b, N)
    return _gemm(a, bm, ldb, False, c, residual, variant)


def linear_into(a: torch.Tensor, w: torch.Tensor, c: torch.Tensor, residual: torch.Tensor | None = None,
                variant: str = "blocked") -> torch.Tensor:
    """c = a @ w^T (+ residual) for an nn.Linear-layout weight w: [N, K]."""
    K = a.shape[1]
    wm, ldw = _row_major(w, K)
    return _gemm(a, wm, ldw, True, c, residual, variant)


GATE_UP_GROUP = 32  # rows of Wg, then of Wu, per group of the packed gate/up weight


def pack_gate_up(wg: torch.Tensor, wu: torch.Tensor) -> torch.Tensor:
    """The [2N, K] weight ``gemm_swiglu_into`` takes: the rows of Wg and Wu
    ([N, K] each, nn.Linear layout) interleaved in groups of 32."""
    if wg.shape != wu.shape or wg.dim() != 2:
        raise ValueError(f"pack_gate_up: Wg {tuple(wg.shape)} and Wu {tuple(wu.shape)} must be equal 2-D shapes")
    N, K = wg.shape
    if N % GATE_UP_GROUP:
        raise ValueError(f"pack_gate_up: N={N} must be a multiple of {GATE_UP_GROUP}")
    g = wg.reshape(N // GATE_UP_GROUP, GATE_UP_GROUP, K)
    u = wu.reshape(N // GATE_UP_GROUP, GATE_UP_GROUP, K)
    return torch.stack((g, u), dim=1).reshape(2 * N, K).contiguous()


def gemm_swiglu_into(a: torch.Tensor, w_gu: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
    """c = silu(a @ Wg^T) * (a @ Wu^T) in one GEMM (model.py:88's gate, up and
    SwiGLU), for bf16 (or fp16) a [M, K], the packed weight w_gu =
    pack_gate_up(Wg, Wu) [2N, K] and c [M, N], all of one dtype.  Equal to two
    linear_into calls in that dtype and a SwiGLU in that dtype."""
    M, K = a.shape
    N = c.shape[1]
    if c.shape[0] != M:
        raise ValueError(f"gemm_swiglu_into: output {tuple(c.shape)} does not have the {M} rows of a")
    if w_gu.shape != (2 * N, K):
        raise ValueError(f"gemm_swiglu_into: packed weight {tuple(w_gu.shape)} does not match [2*{N}, {K}]")
    if not (a.dtype == w_gu.dtype == c.dtype) or a.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("gemm_swiglu_into: bf16 or fp16 operands, all of one dtype")
    a, lda = _row_major(a, K)
    wm, ldw = _row_major(w_gu, K)
    if c.dim() != 2 or (c.stride(1) != 1 and N > 1) or (M > 1 and c.stride(0) < N):
        raise ValueError("gemm_swiglu_into: the output must be a row-major [M, N] tensor")
    ldc = c.stride(0) if M > 1 else max(N, 1)
    _lib.call("nkl_gemm_swiglu", ptr(a), ptr(wm), ptr(c), M, N, K, lda, ldw, ldc, dtype_code(a.dtype),
              stream_handle())
    return c


FP32_SPLIT_K = 1505  # the shortest K nkl_gemm_ws splits over workgroups in fp32 (48 K-steps of 32, begun)


def _splits_k(a: torch.Tensor, w: torch.Tensor, M: int, N: int, K: int) -> bool:
    """Whether a @ w^T splits its K over workgroups.  The one gate/up GEMM does
    not, and its longer sums cost precision there (16 x 4064 x 2048: 23.5 us
    against 28.5, but 5.9e-7 against 4.2e-7 from 64 bits)."""
    return _lib.lib().nkl_gemm_workspace_bytes(a.data_ptr(), w.data_ptr(), M, N, K, a.stride(0), w.stride(0), 1, _lib.F32,
                                               _lib.F32) > 0


def gate_up_into(a: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
    """c = silu(a @ wg^T) * (a @ wu^T) (model.py:88) for a [M, K], nn.Linear-layout
    weights wg, wu [N, K] and c [M, N], all of one dtype: one fp32 GEMM where its
    16-byte accesses fit the operands, else two ``linear_into`` and a SwiGLU."""
    M, K = a.shape
    N = c.shape[1]
    if c.shape[0] != M or wg.shape != (N, K) or wu.shape != (N, K):
        raise ValueError(f"gate_up_into: a {tuple(a.shape)}, Wg {tuple(wg.shape)}, Wu {tuple(wu.shape)} and output "
                         f"{tuple(c.shape)} do not match")
    if (a.dtype == wg.dtype == wu.dtype == c.dtype == torch.float32 and M > 0 and K > 0
            and a.stride(1) == wg.stride(1) == wu.stride(1) == c.stride(1) == 1
            and (K < FP32_SPLIT_K or not _splits_k(a, wg, M, N, K))):
        rc = _lib.lib().nkl_gemm_gate_up(a.data_ptr(), wg.data_ptr(), wu.data_ptr(), c.data_ptr(), M, N, K, a.stride(0),
                                         wg.stride(0), wu.stride(0), c.stride(0), _lib.F32, stream_handle())
        if rc == 0:
            return c
        if rc != _lib.EINVAL:
            _lib.check("nkl_gemm_gate_up", rc)
    gate, up = (torch.empty((M, N), dtype=c.dtype, device=c.device) for _ in range(2))
    linear_into(a, wg, gate)
    linear_into(a, wu, up)
    if not c.is_contiguous():
        return c.copy_(swiglu_into(gate, up, torch.empty_like(gate)))
    return swiglu_into(gate, up, c)


def matmul(a, b, variant: str = "blocked"):
    """C = A @ B for any shapes (ops.py:38-52).  bf16 inputs accumulate in fp32 and
    C is rounded once; the output dtype is the input dtype."""
    M, K = a.shape
    K2, N = b.shape
    assert K == K2, (a.shape, b.shape)
    if variant not in _MATMUL_VARIANTS:
        raise ValueError(f"unknown matmul variant {variant!r}; expected one of {sorted(_MATMUL_VARIANTS)}")
    ta, kind = to_device(a)
    tb, _ = to_device(b)
    if ta.dtype != tb.dtype:
        raise TypeError(f"matmul operands must share a dtype, got {ta.dtype} and {tb.dtype}")
    c = ta.new_empty((M, N))
    gemm_into(ta, tb, c, variant=variant)
    return from_device(c, kind)


def split_bf16_into(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """y[:, :K] = bf16(x), y[:, K:] = bf16(x - y[:, :K]) for an fp32 x [M, K] and a
    bf16 y [M, 2K]: the hi/lo pair a bf16 GEMM against ``stack_k(w)``
    multiplies with fp32 accuracy."""
    if x.dim() != 2 or y.dim() != 2 or y.shape != (x.shape[0], 2 * x.shape[1]):
        raise ValueError(f"split_bf16_into: y {tuple(y.shape)} must be [M, 2K] for x {tuple(x.shape)}")
    if x.dtype != torch.float32 or y.dtype != torch.bfloat16:
        raise TypeError("split_bf16_into: fp32 x and bf16 y expected")
    M, K = x.shape
    x2, _, _, ldx = _as_rows(x)
    if y.stride(1) != 1:
        raise ValueError("split_bf16_into: y must have unit column stride")
    _lib.call("nkl_split_bf16", ptr(x2), ptr(y), M, K, ldx, y.stride(0) if M > 1 else 2 * K, stream_handle())
    return y


def stack_k(w: torch.Tensor) -> torch.Tensor:
    """[w | w] along K for an nn.Linear weight w [N, K] (bf16): the B operand
    that pairs with split_bf16_into's [hi | lo] activations."""
    return torch.cat((w, w), dim=1).contiguous()


# ------------------------------------------------------- 4-bit weights --

@dataclass(frozen=True)
class W4Weight:
    """A weight [n, k] in 4 bits as the kernels take it (``pack_w4``): W[n, k] =
    scale[n, g] * (code[n, k] - zero[n, g]), g = k // group.  paired: a gate and
    an up weight, both [n, k] (``pair_w4``)."""
    packed: torch.Tensor         # int32 [tiles of 16 rows, chunks of 128 columns, 64, 4]
    scales: torch.Tensor         # [tiles, groups, 16]
    zeros: torch.Tensor | None   # uint8 [tiles, groups, 16]; None: 8 throughout
    n: int
    k: int
    group: int
    paired: bool = False

    def __post_init__(self):
        _w4_group("W4Weight", self.group)
        Kc = -(-self.k // 128)
        tiles = -(-self.n // 16) * (2 if self.paired else 1)
        groups = Kc * (128 // self.group) if self.group < 128 else -(-self.k // self.group)
        shapes = {"packed": (self.packed, torch.int32, (tiles, Kc, 64, 4)),
                  "scales": (self.scales, self.scales.dtype, (tiles, groups, 16)),
                  "zeros": (self.zeros, torch.uint8, (tiles, groups, 16))}
        dtype_code(self.scales.dtype)
        for name, (t, dt, shape) in shapes.items():
            if t is not None and (t.shape != shape or t.dtype is not dt or not t.is_contiguous() or t.device != self.packed.device):
                raise ValueError(f"W4Weight: {name} must be a contiguous {dt} {list(shape)} with the packed codes, got "
                                 f"{t.dtype} {list(t.shape)} on {t.device}")


def _w4_group(fn: str, group: int) -> None:
    if group not in (32, 64) and (group < 128 or group % 128):
        raise ValueError(f"{fn}: group={group}; 32, 64 or a multiple of 128 columns expected")


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, group: int = 128) -> W4Weight:
    """Lays out 4-bit codes (uint8 [N, K], 0 .. 15) with a scale for each row and
    `group` columns (fp32, bf16 or fp16 [N, ceil(K / group)]) and zeros (the
    codes that stand for 0: uint8, as scales; None: 8).  Once per weight."""
    fn = "pack_w4"
    _w4_group(fn, group)
    if codes.dim() != 2 or codes.dtype is not torch.uint8 or 0 in codes.shape:
        raise ValueError(f"{fn}: codes must be uint8 [N, K], got {codes.dtype} {list(codes.shape)}")
    N, K = codes.shape
    G = -(-K // group)
    dtype_code(scales.dtype)
    if scales.shape != (N, G) or (zeros is not None and (zeros.shape != (N, G) or zeros.dtype is not torch.uint8)):
        raise ValueError(f"{fn}: scales {list(scales.shape)} and zeros (uint8) must be [{N}, {G}]")
    if int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15):
        raise ValueError(f"{fn}: codes and zeros must lie within 0 .. 15")
    Nt, Kc = -(-N // 16), -(-K // 128)
    c = torch.nn.functional.pad(codes, (0, 128 * Kc - K, 0, 16 * Nt - N))
    # [tile, row, chunk, word, lane group, code] -> [tile, chunk, lane group, row, word, code]
    c = c.view(Nt, 16, Kc, 4, 4, 8).permute(0, 2, 4, 1, 3, 5).reshape(Nt, Kc, 64, 4, 8)
    words = torch.zeros((Nt, Kc, 64, 4), dtype=torch.int64, device=c.device)
    for j in range(8):
        words |= c[..., j].to(torch.int64) << (4 * (j // 2) + 16 * (j % 2))
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    groups = Kc * (128 // group) if group < 128 else G
    tiles = lambda t: (torch.nn.functional.pad(t, (0, groups - G, 0, 16 * Nt - N))  # noqa: E731
                       .view(Nt, 16, groups).transpose(1, 2).contiguous())
    return W4Weight(words, tiles(scales), None if zeros is None else tiles(zeros), N, K, group)


def quantize_w4(w: torch.Tensor, group: int = 128, zeros: bool = False, scale_dtype: torch.dtype | None = None) -> W4Weight:
    """A weight [N, K] in 4 bits: each row's groups scaled so that their largest
    values keep their places (with zeros: the least and largest of them and 0), and
    rounded to the nearest code.  Scales of scale_dtype (w's); 0 for groups of zeros."""
    fn = "quantize_w4"
    _w4_group(fn, group)
    if w.dim() != 2 or 0 in w.shape:
        raise ValueError(f"{fn}: w {tuple(w.shape)} must be [N, K]")
    N, K = w.shape
    sdt = w.dtype if scale_dtype is None else scale_dtype
    dtype_code(sdt)
    G = -(-K // group)
    x = torch.nn.functional.pad(w.detach().float(), (0, G * group - K)).view(N, G, group)
    hi, lo = x.amax(dim=2).clamp(min=0), x.amin(dim=2).clamp(max=0)
    need = (hi - lo) / 15 if zeros else torch.maximum(hi / 7, lo / -8)
    s = need.to(sdt)
    if not bool(torch.isfinite(s).all()):
        raise ValueError(f"{fn}: w holds values that are not finite, or whose scale is none of {sdt}")
    # Subnormal numbers are far apart, and what a scale rounded down to one leaves out is no
    # rounding of the codes: the next larger one (whose bits are the next whole number).
    bits = s.view(torch.int32 if sdt is torch.float32 else torch.int16)
    top, low, sd = hi.double(), -lo.double(), s.double()
    short = top + low > 15 * sd if zeros else (top > 7 * sd) | (low > 8 * sd)
    s = (bits + (short & (s < torch.finfo(sdt).smallest_normal)).to(bits.dtype)).view(sdt)
    sf = torch.where(s != 0, s, torch.ones_like(s)).float()  # (0: of zeros, whose products are then exactly 0)
    z = (-lo / sf).round().clamp(0, 15) if zeros else torch.full_like(sf, 8.0)
    q = ((x / sf[:, :, None]).round() + z[:, :, None]).clamp(0, 15).to(torch.uint8)
    return pack_w4(q.view(N, G * group)[:, :K], s, z.to(torch.uint8) if zeros else None, group)


def pair_w4(gate: W4Weight, up: W4Weight) -> W4Weight:
    """The weight that ``linear_w4_swiglu_into`` takes: the tiles of two weights
    of one shape, group and scale dtype in turn."""
    a, b = ((w.n, w.k, w.group, w.scales.dtype, w.zeros is None, w.paired) for w in (gate, up))
    if a != b or gate.paired:
        raise ValueError(f"pair_w4: weights of (n, k, group, scales' dtype, no zeros, paired) {a} and {b}")
    mix = lambda s, t: torch.stack((s, t), dim=1).reshape(-1, *s.shape[1:])  # noqa: E731
    return W4Weight(mix(gate.packed, up.packed), mix(gate.scales, up.scales),
                    None if gate.zeros is None else mix(gate.zeros, up.zeros), gate.n, gate.k, gate.group, True)


def unpack_w4(w: W4Weight) -> torch.Tensor:
    """The values of an unpaired weight, fp32 [n, k]."""
    if w.paired:
        raise ValueError("unpack_w4: a pair of weights")
    Nt, Kc = w.packed.shape[:2]
    codes = torch.stack([(w.packed >> (4 * (j // 2) + 16 * (j % 2))) & 15 for j in range(8)], dim=-1)
    codes = codes.view(Nt, Kc, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5).reshape(16 * Nt, 128 * Kc)
    spread = lambda t: (t.transpose(1, 2).reshape(16 * Nt, -1).float()  # noqa: E731
                        .repeat_interleave(w.group, dim=1)[:, :128 * Kc][:w.n, :w.k])
    return (codes[:w.n, :w.k].float() - (8.0 if w.zeros is None else spread(w.zeros))) * spread(w.scales)


def _linear_w4(fn: str, a: torch.Tensor, w: W4Weight, c: torch.Tensor, residual: torch.Tensor | None) -> torch.Tensor:
    sa, sc = a.shape, c.shape
    if len(sa) != 2 or len(sc) != 2 or sa[1] != w.k or sc[0] != sa[0] or sc[1] != w.n:
        raise ValueError(f"{fn}: a {tuple(sa)} and output {tuple(sc)} do not match a weight [{w.n}, {w.k}]")
    M, K = sa
    dt, ds, do = a.dtype, w.scales.dtype, c.dtype
    if (ds is not dt and ds is not torch.float32) or (do is not dt and do is not torch.float32):
        raise TypeError(f"{fn}: scales of {ds} and an output of {do} for activations of {dt}: theirs or float32 expected")
    ta, tc = a.stride(), c.stride()
    if M > 1 and tc[0] < w.n or w.n > 1 and tc[1] != 1:
        raise ValueError(f"{fn}: the output must be a row-major [M, N] tensor")
    if K > 1 and ta[1] != 1 or M > 1 and ta[0] < K:
        a = a.contiguous()
        ta = a.stride()
    pr, ldr = None, 0
    if residual is not None:
        if residual.shape != sc or residual.dtype is not do:
            raise ValueError(f"{fn}: residual {tuple(residual.shape)} {residual.dtype} does not match the output "
                             f"{tuple(sc)} {do}")
        if w.n > 1 and residual.stride(1) != 1 or M > 1 and residual.stride(0) < w.n:
            residual = residual.contiguous()
        pr, ldr = residual.data_ptr(), max(residual.stride(0), 0)
    _on_current_device(fn, a, w.packed, c, residual)
    zeros = w.zeros
    rc = _lib.lib().nkl_gemm_w4(a.data_ptr(), w.packed.data_ptr(), w.scales.data_ptr(),
                                None if zeros is None else zeros.data_ptr(), c.data_ptr(), pr, M, w.n, K, w.group,
                                ta[0], tc[0], ldr, w.paired, dtype_code(dt), dtype_code(ds), dtype_code(do),
                                stream_handle())
    if rc:
        _lib.check("nkl_gemm_w4", rc)
    return c


def linear_w4_into(a: torch.Tensor, w: W4Weight, c: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """c = a @ w^T (+ residual) for a 4-bit weight; a [M, k] of any of the three
    dtypes, c [M, n] (which may be the residual, and not a) of a's or fp32, the
    weight's scales likewise.  The weight's values are not rounded: sums are of codes
    times a in fp32 (of 16-bit a: of 16 + code, put right by the sum of a, and as
    exact as those magnitudes are), scaled group by group, and rounded once.  A
    row of a with an infinity or NaN gives NaN, and one of bf16 that overflows
    in 16 + code, beyond 2^116, may."""
    if w.paired:
        raise ValueError("linear_w4_into: a pair of weights; linear_w4_swiglu_into takes those")
    return _linear_w4("linear_w4_into", a, w, c, residual)


def linear_w4_swiglu_into(a: torch.Tensor, w: W4Weight, c: torch.Tensor) -> torch.Tensor:
    """c = silu(a @ gate^T) * (a @ up^T) for ``pair_w4(gate, up)`` in one pass; the
    products are not rounded between."""
    if not w.paired:
        raise ValueError("linear_w4_swiglu_into: pair_w4's weight expected")
    return _linear_w4("linear_w4_swiglu_into", a, w, c, None)


def linear_w4(a, w: W4Weight):
    """a @ w^T in a new array of a's kind and dtype."""
    t, kind = to_device(a)
    return from_device(linear_w4_into(t, w, t.new_empty((t.shape[0], w.n))), kind)


# ---------------------------------------------------------------- RoPE --

def rope_into(x: torch.Tensor, y: torch.Tensor, base: float = 10000.0, pos0: int = 0) -> torch.Tensor:
    """Rotary position embedding (rotate-half layout) of x [H, S, d] into y
    (which may be x): elements i and i + d/2 of row s rotate by
    (pos0 + s) * base^(-2 i / d).  Any strides along H and S; d contiguous."""
    if x.dim() != 3 or y.shape != x.shape or x.dtype != y.dtype:
        raise ValueError(f"rope_into: x {tuple(x.shape)} and y {tuple(y.shape)} must be equal [H, S, d] tensors")
    H, S, d = x.shape
    for t in (x, y):
        if t.stride(2) != 1 and d > 1:
            raise ValueError("rope_into: the head dim must be contiguous")
    _lib.call("nkl_rope", ptr(x), ptr(y), H, S, d, x.stride(0), x.stride(1), y.stride(0), y.stride(1), int(pos0),
              float(base), dtype_code(x.dtype), stream_handle())
    return y


def rope(x, base: float = 10000.0, pos0: int = 0):
    """RoPE of x [H, S, d] (NumPy or torch); returns a new array of x's kind."""
    tx, kind = to_device(x)
    y = torch.empty_like(tx)
    return from_device(rope_into(tx, y, base, pos0), kind)


@dataclass(frozen=True)
class Rotary:
    """How the elements of a head rotate with their position: pair i of the
    first `dim` elements by position * frequency(i), which is base^(-2 i / dim)
    unless scaled.  Pairs are (i, i + dim / 2), or (2 i, 2 i + 1) interleaved.

    scaling, for contexts `factor` times as long as the `original` one (in
    positions) that a model was trained for:
      "linear"  every frequency divided by factor (position interpolation);
      "base"    the base times factor^(dim / (dim - 2)): the lowest frequency
                divided by factor, the highest kept (the NTK-aware base);
      "parts"   (YaRN's NTK-by-parts) the pairs that turn more than high_turns (32) times over the
                original context kept, those that turn less than low_turns (1)
                times divided by factor, a linear ramp over the pairs' numbers
                between; the rotated elements times 0.1 ln(factor) + 1;
      "bands"   the same with the ramp over the turns themselves (high_turns
                4), and no factor of the elements (Llama's longer contexts).
    magnitude replaces the factor of the rotated elements.

    An object is made once and kept: it holds its table of frequencies."""
    dim: int
    base: float = 10000.0
    interleaved: bool = False
    scaling: str | None = None
    factor: float = 1.0
    original: int = 0
    low_turns: float | None = None
    high_turns: float | None = None
    magnitude: float | None = None

    def __post_init__(self):
        dim, base, factor = self.dim, float(self.base), float(self.factor)
        if dim < 2 or dim % 2 or dim > 2 * _lib.ROTARY_PAIRS:
            raise ValueError(f"Rotary: dim={dim} must be even, within [2, {2 * _lib.ROTARY_PAIRS}]")
        if not (1.0 < base < math.inf):
            raise ValueError(f"Rotary: base={self.base} must be above 1")
        if self.scaling not in (None, "linear", "base", "parts", "bands"):
            raise ValueError(f"Rotary: scaling {self.scaling!r}; one of 'linear', 'base', 'parts', 'bands' expected")
        if not (1.0 <= factor < math.inf) or (self.scaling is None and factor != 1.0):
            raise ValueError(f"Rotary: factor={self.factor} must be at least 1 (and 1 without scaling)")
        freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
        magnitude = 1.0
        if self.scaling == "linear":
            freq = [f / factor for f in freq]
        elif self.scaling == "base" and dim > 2:
            stretched = base * factor ** (dim / (dim - 2))
            freq = [stretched ** (-2.0 * i / dim) for i in range(dim // 2)]
        elif self.scaling in ("parts", "bands"):
            low = 1.0 if self.low_turns is None else float(self.low_turns)
            high = (32.0 if self.scaling == "parts" else 4.0) if self.high_turns is None else float(self.high_turns)
            if self.original < 1 or not (0.0 < low < high < math.inf):
                raise ValueError(f"Rotary: scaling {self.scaling!r} needs the original context ({self.original}) and "
                                 f"0 < low_turns ({low}) < high_turns ({high})")
            if self.scaling == "parts":
                def pair(turns):  # the (fractional) number of the pair that turns so often
                    return dim * math.log(self.original / (2 * math.pi * turns)) / (2 * math.log(base))

                first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), dim - 1)
                kept = [1 - min(1.0, max(0.0, (i - first) / max(last - first, 0.001))) for i in range(dim // 2)]
                if pair(low) < 0:  # (the first pair, too, turns less often)
                    kept = [0.0] * (dim // 2)
                magnitude = 0.1 * math.log(factor) + 1
            else:
                kept = [min(1.0, max(0.0, (self.original * f / (2 * math.pi) - low) / (high - low))) for f in freq]
            freq = [f * k + f / factor * (1 - k) for f, k in zip(freq, kept)]
        if self.magnitude is not None:
            magnitude = float(self.magnitude)
            if not math.isfinite(magnitude):
                raise ValueError(f"Rotary: magnitude={self.magnitude}")
        object.__setattr__(self, "frequencies", tuple(freq))
        object.__setattr__(self, "gain", magnitude)
        object.__setattr__(self, "_packed", _lib.pack_rotary(dim // 2, int(self.interleaved), magnitude, *freq,
                                                             *([0.0] * (_lib.ROTARY_PAIRS - dim // 2))))


def rotary_into(x: torch.Tensor, y: torch.Tensor, rotary: Rotary, positions: torch.Tensor | None = None, pos0: int = 0,
                grad: bool = False) -> torch.Tensor:
    """x [H, S, d] rotated into y (which may be x) as `rotary` says: row s by
    positions[s] (int32 or int64 [S], within 2^31) or pos0 + s.  Elements past
    rotary.dim are copied.  Any strides along H and S; d contiguous; y shares no
    memory with x unless it is x.
    grad: the transposed map, which takes the gradient of y (as x) to x's."""
    fn = "rotary_into"
    if x.dim() != 3 or y.shape != x.shape or x.dtype != y.dtype:
        raise ValueError(f"{fn}: x {tuple(x.shape)} {x.dtype} and y {tuple(y.shape)} {y.dtype} must be equal [H, S, d]")
    H, S, d = x.shape
    sx, sy = x.stride(), y.stride()
    if d > 1 and (sx[2] != 1 or sy[2] != 1):
        raise ValueError(f"{fn}: the head dim must be contiguous")
    wide = 0
    if positions is not None:
        if positions.shape != (S,) or positions.dtype not in (torch.int32, torch.int64) or (S > 1 and positions.stride(0) != 1):
            raise ValueError(f"{fn}: positions must be int32 or int64 [{S}] with unit stride, got {positions.dtype} "
                             f"{list(positions.shape)}")
        if pos0:
            raise ValueError(f"{fn}: either positions or pos0")
        wide = int(positions.dtype is torch.int64)
    _on_current_device(fn, x, y, positions)
    rc = _lib.lib().nkl_rotary_apply(rotary._packed, x.data_ptr(), y.data_ptr(), H, S, d, sx[0], sx[1], sy[0], sy[1],
                                     ptr(positions), wide, int(pos0), int(grad), dtype_code(x.dtype), stream_handle())
    if rc:
        _lib.check("nkl_rotary_apply", rc)
    return y


def rotary(x, rotary: Rotary, positions=None, pos0: int = 0, grad: bool = False):
    """``rotary_into`` a new array of x's kind (NumPy or torch; positions too)."""
    tx, kind = to_device(x)
    if positions is not None and not (isinstance(positions, torch.Tensor) and positions.is_cuda):
        positions = torch.as_tensor(positions).to(tx.device)
    return from_device(rotary_into(tx, torch.empty_like(tx), rotary, positions, pos0, grad), kind)


# ------------------------------------------------------------- row ops --

def _as_rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """View t as [rows, cols] with unit column stride: (t2d, rows, cols, ld)."""
    cols = t.shape[-1] if t.dim() > 0 else 1
    t2 = t.reshape(-1, cols) if t.dim() != 2 else t
    if t2.dim() != 2:
        t2 = t2.contiguous()
    ld, cs = t2.stride()
    if (cs != 1 and cols > 1) or ld < cols:
        t2 = t2.contiguous()
        ld = t2.stride(0)
    rows = t2.shape[0]
    return t2, rows, cols, max(ld, cols) if rows > 1 else max(cols, 1)


def softmax_into(x: torch.Tensor, y: torch.Tensor, fused: bool = True) -> torch.Tensor:
    if y.shape != x.shape or y.dtype != x.dtype:
        raise ValueError(f"softmax_into: y {tuple(y.shape)} {y.dtype} must match x {tuple(x.shape)} {x.dtype}")
    x2, R, D, ldx = _as_rows(x)
    y2, _, _, ldy = _as_rows(y)
    dt = dtype_code(x2.dtype)
    if fused:
        rc = _lib.lib().nkl_softmax(x2.data_ptr(), y2.data_ptr(), R, D, ldx, ldy, dt, stream_handle())
        if rc:
            _lib.check("nkl_softmax", rc)
    else:
        nbytes = _lib.lib().nkl_softmax_unfused_workspace_bytes(R, D)
        ws = workspace(nbytes, x2.device)
        _lib.call("nkl_softmax_unfused", ptr(x2), ptr(y2), ptr(ws), nbytes, R, D, ldx, ldy, dt, stream_handle())
    if y2 is not y and y2.data_ptr() != y.data_ptr():
        y.copy_(y2.view_as(y))
    return y


def softmax(x, fused: bool = True):
    """Row softmax over the last dim (ops.py:55-57).  fused=True: one HBM pass
    (norm.py:65); fused=False: three passes through HBM (norm.py:22)."""
    t, kind = to_device(x)
    return from_device(softmax_into(t, t.new_empty(t.shape), fused=fused), kind)


def rmsnorm_into(x: torch.Tensor, weight: torch.Tensor, y: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """y = x * rsqrt(mean(x^2) + eps) * weight.  The normalised row stays in
    fp32 and is multiplied by the weight in the weight's own dtype (fp32 or
    bf16, independent of x's), then rounded once to y's dtype (x's, or bf16
    for an fp32 x)."""
    if y.shape != x.shape:
        raise ValueError(f"rmsnorm_into: y {tuple(y.shape)} must match x {tuple(x.shape)}")
    x2, R, D, ldx = _as_rows(x)
    if weight.numel() != D:
        raise ValueError(f"rmsnorm_into: weight has {weight.numel()} elements, x rows have {D}")
    if y.stride(-1) != 1 or not y.is_contiguous():
        raise ValueError("rmsnorm_into: output must be contiguous")
    w = weight.contiguous()
    rc = _lib.lib().nkl_rmsnorm_ex(x2.data_ptr(), w.data_ptr(), y.data_ptr(), R, D, ldx, D, float(eps),
                                   dtype_code(x2.dtype), dtype_code(w.dtype), dtype_code(y.dtype), stream_handle())
    if rc:
        _lib.check("nkl_rmsnorm_ex", rc)
    return y


def rmsnorm(x, weight, eps: float = 1e-6):
    """y = x * rsqrt(mean(x^2, -1) + eps) * weight (ops.py:60-61)."""
    t, kind = to_device(x)
    w, _ = to_device(weight)
    return from_device(rmsnorm_into(t, w, t.new_empty(t.shape), eps), kind)


def swiglu_into(gate: torch.Tensor, up: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    if up.shape != gate.shape or y.shape != gate.shape:
        raise ValueError(f"swiglu_into: gate {tuple(gate.shape)}, up {tuple(up.shape)} and y {tuple(y.shape)} "
                         "must have one shape")
    if not (gate.dtype == up.dtype == y.dtype):
        raise TypeError(f"swiglu_into: gate, up and y must share a dtype, got {gate.dtype}, {up.dtype}, {y.dtype}")
    g, u = gate.contiguous(), up.contiguous()
    if not y.is_contiguous():
        raise ValueError("swiglu_into: output must be contiguous")
    rc = _lib.lib().nkl_swiglu(g.data_ptr(), u.data_ptr(), y.data_ptr(), g.numel(), dtype_code(g.dtype),
                               stream_handle())
    if rc:
        _lib.check("nkl_swiglu", rc)
    return y


def swiglu(gate, up):
    """y = silu(gate) * up (ops.py:64-65)."""
    g, kind = to_device(gate)
    u, _ = to_device(up)
    if g.shape != u.shape:
        raise ValueError(f"swiglu: gate {tuple(g.shape)} and up {tuple(u.shape)} differ in shape")
    if g.dtype != u.dtype:
        raise TypeError(f"swiglu: gate and up must share a dtype, got {g.dtype} and {u.dtype}")
    return from_device(swiglu_into(g, u, g.new_empty(g.shape)), kind)


# ------------------------------------------------------------ attention --

@dataclass(frozen=True)
class AttentionVariant:
    """One entry of ATTENTION_VARIANTS: which HIP path serves a reference variant."""
    name: str
    path: str          # "flash" (nkl_flash_attn_causal) or "naive" (nkl_attention_naive)
    reference: str     # the reference kernel it stands for


# The reference's four flash kernels differ only in Trainium engine scheduling
# and are numerically the same online-softmax recurrence; on gfx950 one flash
# kernel serves all four (so they agree bitwise).  "naive" keeps the unfused
# three-pass structure with scores and probabilities in HBM.
ATTENTION_VARIANTS = {
    "naive": AttentionVariant("naive", "naive", "attention.py:35 attention_naive"),
    "flash": AttentionVariant("flash", "flash", "attention.py:155 flash_attention"),
    "flash_kv_resident": AttentionVariant("flash_kv_resident", "flash", "attention.py:179 flash_attention_kv_resident"),
    "flash_balanced": AttentionVariant("flash_balanced", "flash", "attention.py:249 flash_attention_balanced"),
    "flash_pipelined": AttentionVariant("flash_pipelined", "flash", "attention.py:280 flash_attention_pipelined"),
}


# Flash-attention scratch, one pair per (device, stream): a partial-state
# workspace (no initialisation needed) and an arrival-counter array zeroed
# once, which the kernel leaves at zero after every call.  Calls on one stream
# run one after another, so they can share both.  Each is grown when a call
# needs more (the counters are then re-zeroed).  Buffers a call has used are
# never freed: a captured HIP graph may still replay launches that point at
# them, so outgrown ones are kept for the life of the process.
_FLASH_SCRATCH: dict = {}
_FLASH_RETIRED: list = []


def _flash_scratch(ws_bytes: int, counter_bytes: int, dev: torch.device,
                   stream: int) -> tuple[torch.Tensor, torch.Tensor]:
    key = (dev, stream)
    ws, cnt = _FLASH_SCRATCH.get(key, (None, None))
    if ws is None or ws.numel() < ws_bytes:
        if ws is not None:
            _FLASH_RETIRED.append(ws)
        ws = torch.empty(max(ws_bytes, 1 << 20), dtype=torch.uint8, device=dev)
    if cnt is None or cnt.numel() * 4 < counter_bytes:
        if cnt is not None:
            _FLASH_RETIRED.append(cnt)
        cnt = torch.zeros(max(counter_bytes // 4, 4096), dtype=torch.int32, device=dev)
    _FLASH_SCRATCH[key] = (ws, cnt)
    return ws, cnt


# The attention entry points' stride limits (elements): between heads, and
# between rows (32-bit byte offsets within a block of up to 256 rows).
ATTN_MAX_HEAD_STRIDE, ATTN_MAX_ROW_STRIDE = 1 << 24, 1 << 21


def _attn_strides_ok(t: torch.Tensor, E: int) -> bool:
    sh, ss, sd = t.stride()
    return (sd == 1 and t.data_ptr() % 16 == 0 and sh % E == 0 and ss % E == 0
            and 0 <= sh <= ATTN_MAX_HEAD_STRIDE and 0 <= ss <= ATTN_MAX_ROW_STRIDE)


def _attn_operand(t: torch.Tensor, E: int) -> torch.Tensor:
    return t if _attn_strides_ok(t, E) else t.contiguous()


def attention_into(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                   variant: str = "flash_pipelined", scale: float | None = None, window: int | None = None,
                   sinks: int = 0) -> torch.Tensor:
    """Causal attention into o; q, o: [H, S, d] and k, v: [Hkv, S, d] GPU tensors
    (Hkv = H, or a divisor of H for grouped-query attention: query head h reads
    K/V head h // (H / Hkv)), any strides along heads and S (d contiguous).
    d must be a multiple of 8 (bf16) / 4 (fp32).  window and sinks as in
    ``attention``."""
    spec = ATTENTION_VARIANTS[variant]
    H, S, d = q.shape
    Hkv = k.shape[0]
    if k.shape != v.shape or k.shape[1:] != q.shape[1:] or Hkv < 1 or H % Hkv:
        raise ValueError(f"attention_into: k, v {tuple(k.shape)}, {tuple(v.shape)} must be [Hkv, S, d] with Hkv "
                         f"dividing the {H} query heads of q {tuple(q.shape)}")
    if o.shape != q.shape or o.dtype != q.dtype or not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f"attention_into: o {tuple(o.shape)} {o.dtype} must match q {tuple(q.shape)} {q.dtype}, "
                         "and k, v share q's dtype")
    return _attention(q, k, v, o, spec, H, Hkv, S, d, 1.0 / math.sqrt(d) if scale is None else float(scale), window,
                      sinks)


def _attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, spec: AttentionVariant, H: int,
               Hkv: int, S: int, d: int, scale: float, window: int | None = None, sinks: int = 0) -> torch.Tensor:
    """attention_into on shapes and dtypes already checked."""
    if window is not None or sinks:
        return _window_attention(q, k, v, o, spec, H, Hkv, S, d, scale, window, sinks)
    E = 8 if q.element_size() == 2 else 4
    q, k, v = (_attn_operand(t, E) for t in (q, k, v))
    o_ok = _attn_strides_ok(o, E)
    out = o if o_ok else torch.empty((H, S, d), dtype=o.dtype, device=o.device)
    strides = (*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *out.stride()[:2])
    dt = dtype_code(q.dtype)
    gqa = Hkv != H
    if spec.path == "flash":
        L, st = _lib.lib(), stream_handle()
        nbytes = L.nkl_flash_attn_causal_workspace_bytes(H, S, d, dt)
        pw, wb, pc, cb = None, 0, None, 0
        if nbytes:
            ws, cnt = _flash_scratch(nbytes, L.nkl_flash_attn_causal_counter_bytes(H, S, dt), q.device, st)
            pw, wb, pc, cb = ws.data_ptr(), ws.numel(), cnt.data_ptr(), cnt.numel() * 4
        rc = L.nkl_flash_attn_causal_gqa(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), pw, wb, pc, cb,
                                         H, Hkv, S, d, *strides, scale, dt, st)
        if rc:
            _lib.check("nkl_flash_attn_causal_gqa", rc)
    else:
        nbytes = _lib.lib().nkl_attention_naive_workspace_bytes(H, S, dt)
        ws = workspace(nbytes, q.device)
        if gqa:
            _lib.call("nkl_attention_naive_gqa", ptr(q), ptr(k), ptr(v), ptr(out), ptr(ws), nbytes, H, Hkv, S, d,
                      *strides, scale, dt, stream_handle())
        else:
            _lib.call("nkl_attention_naive", ptr(q), ptr(k), ptr(v), ptr(out), ptr(ws), nbytes, H, S, d, *strides,
                      float(scale), dt, stream_handle())
    if out is not o:
        o.copy_(out)
    return o


def _window_sinks(fn: str, window: int | None, sinks: int) -> tuple[int, int]:
    """The C ABI's (window, sinks): 0 for no window."""
    if window is None:
        if sinks:
            raise ValueError(f"{fn}: sinks={sinks} without a window (every key is visible)")
        return 0, 0
    if int(window) < 1 or int(sinks) < 0:
        raise ValueError(f"{fn}: window={window} must be at least 1 and sinks={sinks} at least 0")
    return min(int(window), MAX_ROWS), min(int(sinks), MAX_ROWS)


def _window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, spec: AttentionVariant, H: int,
                      Hkv: int, S: int, d: int, scale: float, window: int | None, sinks: int) -> torch.Tensor:
    """_attention under a window: the paged kernel over one sequence, k and v as its one page."""
    if spec.path != "flash":
        raise ValueError(f"attention: variant {spec.name!r} has no window; one of the flash variants expected")
    w, sinks = _window_sinks("attention", window, sinks)
    _on_current_device("attention", q, k, v, o)
    if S == 0 or H == 0:
        return o
    if d == 0:
        raise ValueError("attention: head dim 0")
    if S > MAX_ROWS:
        raise ValueError(f"attention: {S} positions, at most {MAX_ROWS} under a window")
    E = 16 // q.element_size()
    q, k, v = (_rows_operand(t, E) for t in (q, k, v))
    out = o if _rows_ok(o, E) else torch.empty((H, S, d), dtype=o.dtype, device=o.device)
    desc = _lib.pack_cache(k.data_ptr(), v.data_ptr(), 0, k.stride(0), k.stride(1), 0, v.stride(0), v.stride(1), 0, 0, 0, 0, 1,
                           Hkv, S, d, 1, 1, S, S, dtype_code(q.dtype))
    _paged_attention(desc, q, (q.stride(1), q.stride(0)), out, (out.stride(1), out.stride(0)), H, w, sinks, None, 0, scale)
    if out is not o:
        o.copy_(out)
    return o


def attention(q, k, v, variant: str = "flash_pipelined", scale: float | None = None, window: int | None = None,
              sinks: int = 0):
    """Causal attention. q, k, v: [H, S, d] (ops.py:77-91); scale 1/sqrt(d)
    unless given (the kernel-level entry points of nkilab.kernels.attention
    pass theirs).
    k and v may also have fewer heads Hkv dividing H (grouped-query attention:
    query head h uses K/V head h // (H / Hkv)), which the reference lacks.
    With a window, query i sees the keys j <= i with j > i - window or
    j < sinks (the paged cache's attention over one sequence; the flash
    variants only, scale > 0), which the reference lacks too.

    The reference pads S to a multiple of 128 and transposes q and k on the
    host; the HIP kernels take [H, S, d] as is and bound-check ragged S, so
    neither copy is made.  A head dim that is not a multiple of the 16-byte
    vector width is zero-padded here (zeros change no dot product) and cropped.
    """
    spec = ATTENTION_VARIANTS[variant]  # KeyError for unknown names, as in the reference
    tq, kind = to_device(q)
    tk, _ = to_device(k)
    tv, _ = to_device(v)
    if not (tq.dtype == tk.dtype == tv.dtype):
        raise TypeError("attention: q, k and v must share a dtype")
    if (tq.dim() != 3 or tk.shape != tv.shape or tk.dim() != 3 or tk.shape[1:] != tq.shape[1:]
            or tk.shape[0] < 1 or tq.shape[0] % tk.shape[0]):
        raise ValueError(f"attention: q must be [H, S, d] and k, v [Hkv, S, d] with Hkv dividing H, got "
                         f"{tuple(tq.shape)}, {tuple(tk.shape)}, {tuple(tv.shape)}")
    H, S, d = tq.shape
    assert d <= 128, "head dim must be <= 128"
    E = 8 if tq.element_size() == 2 else 4
    dp = -(-d // E) * E
    if dp != d:
        tq, tk, tv = (torch.nn.functional.pad(t, (0, dp - d)) for t in (tq, tk, tv))
    o = tq.new_empty((H, S, dp))
    _attention(tq, tk, tv, o, spec, H, tk.shape[0], S, dp, 1.0 / math.sqrt(d) if scale is None else float(scale),
               window, sinks)
    if dp != d:
        o = o[:, :, :d].contiguous()
    return from_device(o, kind)


# ---------------------------------------------------------- paged cache --

MAX_ROWS = 1 << 30  # rows a page table addresses at most, and new rows of a call
E4M3 = torch.float8_e4m3fn  # codes of a cache in 8 bits
ACCEPT8_NODES = 1024  # nodes of a path that is accepted in one


def _cache_code(dt: torch.dtype) -> int:
    return _lib.E4M3 if dt is E4M3 else dtype_code(dt)


def _scales(fn: str, k_cache: torch.Tensor, k_scale: torch.Tensor | None, v_scale: torch.Tensor | None) -> bytes | None:
    """The C ABI's description of the scales of a cache in 8 bits (None: of another), checked."""
    if k_cache.dtype is not E4M3:
        if k_scale is not None or v_scale is not None:
            raise ValueError(f"{fn}: scales belong to a cache of {E4M3}, this one is of {k_cache.dtype}")
        return None
    want = k_cache.shape[:-2]
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t is None or t.dtype is not torch.uint8 or t.shape != want:
            raise ValueError(f"{fn}: {name} must be uint8 {list(want)}, the exponents of a cache of {E4M3}; got "
                             f"{None if t is None else (t.dtype, list(t.shape))}")
    sk, sv = k_scale.stride(), v_scale.stride()
    return _lib.pack_scales(k_scale.data_ptr(), v_scale.data_ptr(), sk[-2], sk[-1], sv[-2], sv[-1])


@lru_cache(maxsize=64)
def _rope(d: int, base: float) -> "Rotary":
    """The table that a rotary base stands for."""
    return Rotary(d, base)


def _rows_ok(t: torch.Tensor, E: int) -> bool:
    """Whether the paged kernels take t [., ., d] as it lies: a row's elements together, rows on 16 bytes."""
    a, b, c = t.stride()
    return c == 1 and a % E == 0 and b % E == 0 and a >= 0 and b >= 0 and t.data_ptr() % 16 == 0


def _rows_operand(t: torch.Tensor, E: int) -> torch.Tensor:
    return t if _rows_ok(t, E) else t.clone(memory_format=torch.contiguous_format)


def _on_current_device(fn: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    """The kernels run on the current device's current stream: every tensor has to be there."""
    d = first.get_device()
    if d >= 0 and d == current_device():
        for t in others:
            if t is not None and t.get_device() != d:
                break
        else:
            return
    raise ValueError(f"{fn}: tensors on {sorted({str(t.device) for t in (first, *others) if t is not None})}, every one "
                     "must be on the current device")


def _int32(fn: str, name: str, t: torch.Tensor, shape: tuple) -> None:
    if t.dtype is not torch.int32 or t.shape != shape or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{fn}: {name} must be int32 {list(shape)} with unit stride, got {t.dtype} {list(t.shape)}")


def _cache_tensors(fn: str, k_cache: torch.Tensor, v_cache: torch.Tensor, layers: bool = False) -> tuple:
    """(shape, k's strides, v's strides) of a cache's tensors, checked."""
    shape, sk, sv = k_cache.shape, k_cache.stride(), v_cache.stride()
    n = len(shape)
    if (n != 4 and not (layers and n == 5)) or shape != v_cache.shape or k_cache.dtype is not v_cache.dtype:
        raise ValueError(f"{fn}: k_cache {tuple(shape)} {k_cache.dtype} and v_cache {tuple(v_cache.shape)} "
                         f"{v_cache.dtype} must be equal {'[layers,] ' if layers else ''}[pages, kv_heads, page_size, d]")
    if (sk[-1] != 1 or sv[-1] != 1) and shape[-1] > 1:
        raise ValueError(f"{fn}: the caches' head dim must be contiguous")
    return shape, sk, sv


def _cache_desc(fn: str, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor,
                q_start: torch.Tensor | None, rows: int, max_q: int | None) -> tuple[bytes, torch.Size, int]:
    """The C ABI's description of a cache and a call's new rows (checked), the cache's shape, and max_new."""
    shape, sk, sv = _cache_tensors(fn, k_cache, v_cache)
    pages, Hkv, page_size, d = shape
    ts = page_table.shape
    if len(ts) != 2:
        raise ValueError(f"{fn}: page_table must be [batch, pages of a sequence], got {tuple(ts)}")
    B, cols = ts
    # (the checks of _int32, called where one fails)
    if page_table.dtype is not torch.int32 or (cols > 1 and page_table.stride(1) != 1):
        _int32(fn, "page_table", page_table, ts)
    ls = lens.shape
    if lens.dtype is not torch.int32 or len(ls) != 1 or ls[0] != B or (B > 1 and lens.stride(0) != 1):
        _int32(fn, "lens", lens, (B,))
    pstart = 0
    if q_start is not None:
        ls = q_start.shape
        if q_start.dtype is not torch.int32 or len(ls) != 1 or ls[0] != B + 1 or (B > 0 and q_start.stride(0) != 1):
            _int32(fn, "q_start", q_start, (B + 1,))
        if max_q is None:
            raise ValueError(f"{fn}: q_start needs max_q, the most new rows of a sequence")
        pstart = q_start.data_ptr()
    else:
        each = rows // B if B else 0
        if each * B != rows:
            raise ValueError(f"{fn}: {rows} rows are not a number for each of {B} sequences; q_start expected")
        if max_q is not None and max_q != each:
            raise ValueError(f"{fn}: max_q={max_q}, and {each} rows for each sequence")
        max_q = each
    if max_q < 0:
        raise ValueError(f"{fn}: max_q={max_q} is negative")
    max_q = min(int(max_q), rows)
    return _lib.pack_cache(k_cache.data_ptr(), v_cache.data_ptr(), sk[0], sk[1], sk[2], sv[0], sv[1], sv[2],
                           page_table.data_ptr() if cols else lens.data_ptr(),  # (no columns: any address, never read)
                           page_table.stride(0), lens.data_ptr(), pstart, pages, Hkv, page_size, d, cols, B, rows, max_q,
                           _cache_code(k_cache.dtype)), shape, max_q


def _tree_words(fn: str, tree: torch.Tensor | None, rows: int, max_q: int) -> tuple[int | None, int]:
    if tree is None:
        return None, 0
    if tree.dtype != torch.int64 or tree.dim() != 2 or tree.shape[0] != rows or 64 * tree.shape[1] < max_q:
        raise ValueError(f"{fn}: tree must be int64 [{rows}, words of 64 nodes for up to {max_q}], got {tree.dtype} "
                         f"{list(tree.shape)}")
    if not tree.is_contiguous():
        raise ValueError(f"{fn}: tree must be contiguous")
    return tree.data_ptr(), tree.shape[1]


def tree_mask(parents: torch.Tensor, q_start: torch.Tensor | None = None, max_q: int | None = None, batch: int = 1,
              window: int | None = None, sinks: int = 0, lens: torch.Tensor | None = None) -> torch.Tensor:
    """Mask words [rows, words] (int64, bit i % 64 of word i // 64 for node i) of
    drafted trees: node t sees itself and its ancestors.  parents: int32 [rows],
    each node's parent as an index within its own sequence's nodes, below the
    node's (-1: a root, which hangs off the context).  q_start: int32
    [batch + 1], the sequences' first rows, with max_q their most nodes;
    without it, rows / batch nodes each.

    With a window a node sees, of its ancestors, those whose positions lie
    within `window` of its own, and those at positions below `sinks` (which
    takes lens: int32 [batch], each sequence's rows with its nodes).
    ``paged_attention`` takes new rows by their bits, so trees deeper than its
    window take these words; ``cache_append_into``, which counts a node's depth
    in them, takes the words without a window."""
    fn = "tree_mask"
    rows = parents.shape[0] if parents.dim() == 1 else -1
    _int32(fn, "parents", parents, (rows,))
    each = 0
    if q_start is not None:
        batch = q_start.shape[0] - 1 if q_start.dim() == 1 else -1
        _int32(fn, "q_start", q_start, (batch + 1,))
        if batch < 0 or max_q is None or int(max_q) < 0:
            raise ValueError(f"{fn}: q_start [batch + 1] and max_q, the most nodes of a sequence, expected")
    else:
        each = rows // batch if batch > 0 else 0
        if each * batch != rows or (max_q is not None and int(max_q) != each):
            raise ValueError(f"{fn}: {rows} nodes are not a number (max_q={max_q}) for each of {batch} sequences")
        max_q = each
    window, sinks = _window_sinks(fn, window, sinks)
    if sinks:
        if lens is None:
            raise ValueError(f"{fn}: sinks need lens, the sequences' rows")
        _int32(fn, "lens", lens, (batch,))
    _on_current_device(fn, parents, q_start, lens)
    # (rows that belong to no sequence see nothing)
    words = (torch.empty if q_start is None else torch.zeros)((rows, max(1, -(-int(max_q) // 64))), dtype=torch.int64,
                                                              device=parents.device)
    _lib.call("nkl_tree_mask_window", ptr(parents), ptr(q_start), ptr(lens), batch, rows, each, window, sinks, ptr(words),
              words.shape[1], stream_handle())
    return words


def cache_append_into(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      page_table: torch.Tensor, lens: torch.Tensor, q_start: torch.Tensor | None = None,
                      max_q: int | None = None, tree: torch.Tensor | None = None, q: torch.Tensor | None = None,
                      q_out: torch.Tensor | None = None, rope_base: float | None = None, rotary: "Rotary | None" = None,
                      k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """Writes new K and V rows (k, v: [rows, kv_heads, d]) to a paged cache
    (k_cache, v_cache: [pages, kv_heads, page_size, d], any strides, d
    contiguous), in one launch with their rotary embedding.

    page_table: int32 [batch, columns], the pages of each sequence in order;
    entries outside [0, pages) name none.  lens: int32 [batch], each sequence's
    rows with the new ones, which are its last.  q_start: int32 [batch + 1],
    the sequences' first new rows, with max_q the most of one (None:
    rows / batch each).  A row that has no place is not written.

    With rope_base, K rows are rotated by their positions on the way (and q
    [rows, H, d] into q_out, which may be q): rotate-half layout, angles in 64
    bits.  tree (``tree_mask``'s words): a node's position is the context's
    length and its depth.  Sequences of one call must not share a page that
    either writes.

    rotary (in rope_base's place): any ``Rotary`` of the head; angles in 64 bits,
    rows rotated in fp32 (what becomes codes in 64 bits) and rounded once.

    A cache in 8 bits (float8_e4m3fn, d and strides multiples of 16) takes rows
    of any of the three dtypes, and k_scale and v_scale, uint8 [pages,
    kv_heads]: a value is its code times 2^(scale - 127), the scale its page's and
    head's.  A page gets the smallest scale with which its rows stay within
    448; where that rises with the new rows, the codes of the rows before
    them follow (rounded again only where they become subnormal).  It does not
    fall again when rows are dropped: a rejected draft can cost kept rows bits."""
    fn = "cache_append_into"
    ks = k.shape
    if len(ks) != 3 or ks != v.shape:
        raise ValueError(f"{fn}: k {tuple(ks)} and v {tuple(v.shape)} must be equal [rows, kv_heads, d]")
    rows, Hkv, d = ks
    desc, shape, max_new = _cache_desc(fn, k_cache, v_cache, page_table, lens, q_start, rows, max_q)
    if Hkv != shape[1] or d != shape[3]:
        raise ValueError(f"{fn}: k {tuple(ks)} must be [rows, kv_heads, d] of the caches {tuple(shape)}")
    dt = k.dtype
    scales = _scales(fn, k_cache, k_scale, v_scale)
    if v.dtype is not dt or (scales is None and k_cache.dtype is not dt):
        raise TypeError(f"{fn}: k {dt}, v {v.dtype} and the caches {k_cache.dtype} must share a dtype")
    if rotary is not None and rope_base is not None:
        raise ValueError(f"{fn}: either rope_base or rotary")
    words, nwords = _tree_words(fn, tree, rows, max_new)
    base = 0.0
    if rope_base is not None:
        base = float(rope_base)
        if not base > 1.0:
            raise ValueError(f"{fn}: rope_base {rope_base} must be above 1")
    sk, sv = k.stride(), v.stride()
    packed = d < 2 or (sk[2] == 1 and sv[2] == 1)
    H, sq, so, pq, po = 0, (0, 0, 1), (0, 0, 1), None, None
    if q is not None or q_out is not None:
        if (rope_base is None and rotary is None) or q is None or q_out is None:
            raise ValueError(f"{fn}: q, q_out and rope_base or rotary go together")
        qs = q.shape
        if len(qs) != 3 or qs != q_out.shape or qs[0] != rows or qs[2] != d:
            raise ValueError(f"{fn}: q {tuple(qs)} and q_out {tuple(q_out.shape)} must be [{rows}, H, {d}]")
        if q.dtype is not dt or q_out.dtype is not dt:
            raise TypeError(f"{fn}: q {q.dtype} and q_out {q_out.dtype} must have k's dtype {dt}")
        H = qs[1]
        if H:
            sq, so, pq, po = q.stride(), q_out.stride(), q.data_ptr(), q_out.data_ptr()
            packed = packed and (d < 2 or (sq[2] == 1 and so[2] == 1))
    if not packed:
        raise ValueError(f"{fn}: the head dim must be contiguous")
    _on_current_device(fn, k, v, k_cache, v_cache, page_table, lens, q_start, tree, q, q_out)
    if scales is not None or rotary is not None:
        if scales is not None:
            _on_current_device(fn, k_scale, v_scale)
        if rotary is None and rope_base is not None:
            rotary = _rope(d, base)
        rc = _lib.lib().nkl_cache_write(desc, scales, k.data_ptr(), v.data_ptr(), sk[0], sk[1], sv[0], sv[1], pq, po, H,
                                        sq[0], sq[1], so[0], so[1], words, nwords,
                                        None if rotary is None else rotary._packed, dtype_code(dt), stream_handle())
        if rc:
            _lib.check("nkl_cache_write", rc)
        return
    rc = _lib.lib().nkl_cache_append(desc, k.data_ptr(), v.data_ptr(), sk[0], sk[1], sv[0], sv[1], pq, po, H, sq[0], sq[1],
                                     so[0], so[1], words, nwords, base, stream_handle())
    if rc:
        _lib.check("nkl_cache_append", rc)


def _layer_desc(fn: str, k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple:
    """(layers, layer strides, [pages, kv_heads, page_size, d], its strides in both) of caches with or without layers."""
    shape, sk, sv = _cache_tensors(fn, k_cache, v_cache, layers=True)
    if len(shape) == 5:
        return shape[0], sk[0], sv[0], shape[1:], sk[1:], sv[1:]
    return 1, 0, 0, shape, sk, sv


def cache_copy_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, pairs, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> None:
    """Copies pages of a cache ([pages, kv_heads, page_size, d], or with a
    leading axis of layers, in each): pairs is a list of (from, to) page ids on
    the host (or an integer array [n, 2]).  A page that is written twice, or
    both read and written, is refused.  Of a cache in 8 bits the scales
    ([layers,] pages, kv_heads) are copied with it."""
    fn = "cache_copy_pages"
    layers, kl, vl, shape, sk, sv = _layer_desc(fn, k_cache, v_cache)
    scales = _scales(fn, k_cache, k_scale, v_scale)
    if isinstance(pairs, torch.Tensor) and pairs.is_cuda:
        raise ValueError(f"{fn}: pairs are read on the host: a list, an array or a CPU tensor expected")
    try:  # (packed by struct: a thousand pairs in a third of the time that an array made of them takes)
        if isinstance(pairs, (list, tuple)):
            flat = list(chain.from_iterable(pairs))
            whole = not pairs or set(map(len, pairs)) == {2}
        else:
            p = np.asarray(pairs)
            whole = p.size == 0 or (p.ndim == 2 and p.shape[1] == 2 and p.dtype.kind in "iu")
            flat = p.ravel().tolist()
        ids = struct.pack(f"{len(flat)}i", *flat)
    except (TypeError, struct.error):
        whole = False
    if not whole:
        raise ValueError(f"{fn}: pairs must be whole numbers [n, 2]")
    if not flat:
        return
    if len(flat) < 64:
        low, high = min(flat), max(flat)
    else:
        view = np.frombuffer(ids, np.int32)
        low, high = int(view.min()), int(view.max())
    if low < 0 or high >= shape[0]:
        raise ValueError(f"{fn}: pages {low} .. {high} outside [0, {shape[0]})")
    _on_current_device(fn, k_cache, v_cache, k_scale, v_scale)
    desc = _lib.pack_cache(k_cache.data_ptr(), v_cache.data_ptr(), sk[0], sk[1], sk[2], sv[0], sv[1], sv[2], 0, 0, 0, 0,
                           *shape, 0, 0, 0, 0, _cache_code(k_cache.dtype))
    rc = _lib.lib().nkl_cache_copy_pages(desc, ids, len(flat) // 2, layers, kl, vl, stream_handle())
    if rc == 0 and scales is not None:  # the scales as a cache of one-byte rows
        tk, tv = k_scale.stride(), v_scale.stride()
        desc = _lib.pack_cache(k_scale.data_ptr(), v_scale.data_ptr(), tk[-2], tk[-1], 0, tv[-2], tv[-1], 0, 0, 0, 0, 0,
                               shape[0], shape[1], 1, 1, 0, 0, 0, 0, _lib.E4M3)
        rc = _lib.lib().nkl_cache_copy_pages(desc, ids, len(flat) // 2, layers, tk[0] if len(tk) == 3 else 0,
                                             tv[0] if len(tv) == 3 else 0, stream_handle())
    if rc:
        _lib.check("nkl_cache_copy_pages", rc)


def cache_accept(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor,
                 paths: torch.Tensor, q_start: torch.Tensor | None = None, n_nodes: int | None = None,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Keeps the accepted path of each sequence's newest rows (the nodes of a
    drafted tree): row paths[b, i] of them moves to row i, in every layer of
    the caches ([layers,] pages, kv_heads, page_size, d), and the sequence's
    new length is returned (int32 [batch], lens unchanged).

    lens: int32 [batch], rows with the nodes.  paths: int32 [batch, columns],
    strictly ascending nodes, ended by the first entry that is not (-1 by
    custom).  The nodes of each sequence: q_start (int32 [batch + 1]), or
    n_nodes for every one.  No other sequence may have a page that rows are
    moved to (those that they come from are only read).

    In a cache of 8 bits (with its scales, [layers,] pages, kv_heads; paths of at
    most 1024 columns) a page that rows move to gets the largest scale of those
    it then holds rows of, and its codes follow."""
    fn = "cache_accept"
    layers, kl, vl, shape, sk, sv = _layer_desc(fn, k_cache, v_cache)
    scales = _scales(fn, k_cache, k_scale, v_scale)
    ts, ps = page_table.shape, paths.shape
    if len(ts) != 2 or len(ps) != 2:
        raise ValueError(f"{fn}: page_table {tuple(ts)} and paths {tuple(ps)} must have two axes")
    B = ts[0]
    _int32(fn, "page_table", page_table, ts)
    _int32(fn, "lens", lens, (B,))
    _int32(fn, "paths", paths, (B, ps[1]))
    if (q_start is None) == (n_nodes is None):
        raise ValueError(f"{fn}: either q_start or n_nodes expected")
    pstart = 0
    if q_start is not None:
        _int32(fn, "q_start", q_start, (B + 1,))
        rows = most = MAX_ROWS
        pstart = q_start.data_ptr()
    else:
        most = int(n_nodes)
        rows = most * B
        if most < 0 or rows > MAX_ROWS:
            raise ValueError(f"{fn}: n_nodes={n_nodes} for {B} sequences")
    _on_current_device(fn, k_cache, v_cache, page_table, lens, paths, q_start, k_scale, v_scale)
    out = torch.empty((B,), dtype=torch.int32, device=lens.device)
    desc = _lib.pack_cache(k_cache.data_ptr(), v_cache.data_ptr(), sk[0], sk[1], sk[2], sv[0], sv[1], sv[2],
                           page_table.data_ptr() if ts[1] else lens.data_ptr(), page_table.stride(0), lens.data_ptr(),
                           pstart, *shape, ts[1], B, rows, most,
                           _cache_code(k_cache.dtype))
    if scales is not None:
        five = k_scale.dim() == 3
        rc = _lib.lib().nkl_cache_accept8(desc, scales, paths.data_ptr(), paths.stride(0), ps[1], out.data_ptr(), layers, kl,
                                          vl, k_scale.stride(0) if five else 0, v_scale.stride(0) if five else 0,
                                          stream_handle())
    else:
        rc = _lib.lib().nkl_cache_accept(desc, paths.data_ptr(), paths.stride(0), ps[1], out.data_ptr(), layers, kl, vl,
                                         stream_handle())
    if rc:
        _lib.check("nkl_cache_accept", rc)
    return out


def _paged_attention8(desc: bytes, scales: bytes, q, sq, o, so, H: int, window: int, sinks: int, words: int | None,
                      nwords: int, scale: float) -> None:
    """nkl_paged_attention8 on operands already checked."""
    L, st, dt = _lib.lib(), stream_handle(), dtype_code(q.dtype)
    args = (desc, scales, dt, q.data_ptr(), o.data_ptr(), H, sq[0], sq[1], so[0], so[1], window, sinks, words, nwords, scale)
    # (as below)
    rc = L.nkl_paged_attention8(*args, None, 0, st)
    if rc == _lib.EWORKSPACE:
        nbytes = L.nkl_paged_attention8_workspace_bytes(desc, H, window, sinks, words is not None, dt)
        rc = L.nkl_paged_attention8(*args, workspace(nbytes, q.device).data_ptr(), nbytes, st)
    if rc:
        _lib.check("nkl_paged_attention8", rc)


def _paged_attention(desc: bytes, q, sq, o, so, H: int, window: int, sinks: int, words: int | None, nwords: int,
                     scale: float) -> None:
    """nkl_paged_attention on operands already checked."""
    L, pq, po, st = _lib.lib(), q.data_ptr(), o.data_ptr(), stream_handle()
    # Short calls need no workspace; the call says so before it launches anything.
    rc = L.nkl_paged_attention(desc, pq, po, H, sq[0], sq[1], so[0], so[1], window, sinks, words, nwords, scale, None, 0, st)
    if rc == _lib.EWORKSPACE:
        nbytes = L.nkl_paged_attention_workspace_bytes(desc, H, window, sinks, words is not None)
        ws = workspace(nbytes, q.device)
        rc = L.nkl_paged_attention(desc, pq, po, H, sq[0], sq[1], so[0], so[1], window, sinks, words, nwords, scale,
                                   ws.data_ptr(), nbytes, st)
    if rc:
        _lib.check("nkl_paged_attention", rc)


def paged_attention_into(q: torch.Tensor, o: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         page_table: torch.Tensor, lens: torch.Tensor, q_start: torch.Tensor | None = None,
                         max_q: int | None = None, window: int | None = None, sinks: int = 0,
                         tree: torch.Tensor | None = None, scale: float | None = None, k_scale: torch.Tensor | None = None,
                         v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over a paged cache that holds their K and V rows
    already (``cache_append_into``), into o; q, o: [rows, H, d], H a multiple of
    the caches' kv_heads (query head h reads K/V head h // (H / kv_heads)).
    The cache arguments are those of ``cache_append_into``.

    New row i of n, at position p = lens[b] - n + i, sees the keys j <= p: all
    of them, or with a window those with j > p - window or j < sinks.  With a
    tree (``tree_mask``'s words, or any bits: bit i lets it see new row i) it
    sees those new rows (whatever the window, which ``tree_mask`` takes for trees
    deeper than it), and of the rows before them those in the window of
    position lens[b] - n - 1 + (new rows it sees), and the sinks.  A row that
    sees nothing gets zeros.  Keys a row does not see take no part, whatever
    they hold; pages that no row of the call sees are not read, and may have
    been freed.  Rows of o that belong to no sequence are left as they are.
    d a multiple of 8 (fp32: 4), at most 128; the caches' strides too, and
    their first elements on 16 bytes; scale above 0; at most 65535 sequences.

    A cache in 8 bits comes with k_scale and v_scale (``cache_append_into``); q
    and o are of any of the three dtypes, d and the caches' strides multiples
    of 16.  Codes' values are exact in bf16 and fp32; in fp16 those outside its
    normal numbers are rounded, to 65504 at most."""
    fn = "paged_attention_into"
    qs = q.shape
    if len(qs) != 3 or o.shape != qs or o.dtype is not q.dtype:
        raise ValueError(f"{fn}: q {tuple(qs)} {q.dtype} and o {tuple(o.shape)} {o.dtype} must be equal [rows, H, d]")
    scales = _scales(fn, k_cache, k_scale, v_scale)
    if scales is None and q.dtype is not k_cache.dtype:
        raise TypeError(f"{fn}: q {q.dtype} and the caches {k_cache.dtype} must share a dtype")
    rows, H, d = qs
    desc, shape, max_new = _cache_desc(fn, k_cache, v_cache, page_table, lens, q_start, rows, max_q)
    if d != shape[3] or H < 1 or H % max(shape[1], 1):
        raise ValueError(f"{fn}: q {tuple(qs)} does not match caches {tuple(shape)}")
    window, sinks = _window_sinks(fn, window, sinks)
    words, nwords = _tree_words(fn, tree, rows, max_new)
    if scale is None:
        scale = 1.0 / math.sqrt(d) if d else 1.0
    _on_current_device(fn, q, o, k_cache, v_cache, page_table, lens, q_start, tree, k_scale, v_scale)
    if max_new == 0:
        return o
    E = 16 // q.element_size()
    q = _rows_operand(q, E)
    out = o if _rows_ok(o, E) else o.clone(memory_format=torch.contiguous_format)
    if scales is not None:
        _paged_attention8(desc, scales, q, q.stride(), out, out.stride(), H, window, sinks, words, nwords, float(scale))
    else:
        _paged_attention(desc, q, q.stride(), out, out.stride(), H, window, sinks, words, nwords, float(scale))
    if out is not o:
        o.copy_(out)
    return o


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lens: torch.Tensor, q_start: torch.Tensor | None = None, max_q: int | None = None,
                    window: int | None = None, sinks: int = 0, tree: torch.Tensor | None = None,
                    scale: float | None = None, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention_into`` a new tensor (whose rows that belong to no
    sequence, if there are any, hold nothing of meaning)."""
    return paged_attention_into(q, torch.empty(q.shape, dtype=q.dtype, device=q.device), k_cache, v_cache, page_table,
                                lens, q_start, max_q, window, sinks, tree, scale, k_scale, v_scale)
