"""Operator API of the B200 W4A16 library: weights on the GPU, decode GEMV / skinny GEMM, prefill dequantize.

Drop-in for lowbit/ops.py of YuchenHe985/lowbit-kernels: the same public names, arguments, defaults and
exceptions. What differs is underneath: the kernels are hand-written for sm_100a and reached through a C ABI
(include/lowbit_b200.h, loaded by ``ext()``), layouts are built on the GPU, and the row-count dispatch
constants come from a B200 sweep (dispatch_b200.json).

Kernel versions (``gemv(x, wq, version)``; the reference's numbering, csrc/w4_gemv.cu:1-22):
  1, 2  canonical layout, M <= 8        -- compatibility kernels (fp32 accumulation)
  3, 4  v3 layout, M <= 8               -- compatibility kernels (fp32 accumulation)
  6     mma layout, M <= 8              -- the decode GEMV (tensor-core fragments fed from registers)
  5     mma layout, M <= 64             -- the skinny tensor-core GEMM
"""
import json
import os
import pathlib

import torch

from . import quant
from ._lib import DTYPE_IDS, Ext, _Device

_EXT = None


def ext():
    """The kernel library (built ahead of time by build.py; no JIT, no fallback). Raises if it cannot load."""
    global _EXT
    if _EXT is None:
        _EXT = Ext()
    return _EXT


LAYOUTS = ("canonical", "v3", "mma")


def _to_device_u8(a, device):
    t = a if isinstance(a, torch.Tensor) else torch.from_numpy(a)
    return t.to(device=device, dtype=torch.uint8).contiguous()


def _to_device_f16(a, device):
    t = a if isinstance(a, torch.Tensor) else torch.from_numpy(a)
    return t.to(device=device, dtype=torch.float16).contiguous()


class W4Weight:
    """One linear layer's weight in the lowbit/quant.py format, on the GPU. `layouts` picks which copies to keep:
    canonical (versions 1, 2, dequantize), v3 (3, 4), mma (5, 6, dequantize; K and the group size multiples of
    128). None = every layout this shape supports; a model keeps ("mma",). Prefill dequantizes, so one of
    canonical / mma must be kept. `packed` is the canonical layout as a numpy array or a torch tensor (host or
    GPU); the other layouts are built from it on the GPU (lowbit/ops.py:24-54)."""

    def __init__(self, packed, scales, group, layouts=None, device=None):
        self.group = group
        self.n, self.k = int(packed.shape[0]), int(packed.shape[1]) * 2
        mma_ok = self.k % 128 == 0 and group % 128 == 0
        if layouts is None:
            layouts = LAYOUTS if mma_ok else ("canonical", "v3")
        if not set(layouts) <= set(LAYOUTS):
            raise ValueError(f"unknown layout in {layouts}; choose from {LAYOUTS}")
        if "mma" in layouts and not mma_ok:
            raise ValueError(f"the mma layout needs K and the group size to be multiples of 128 (K={self.k}, G={group})")
        if "canonical" not in layouts and "mma" not in layouts:
            raise ValueError("keep the canonical or the mma layout: prefill dequantizes from one of them")
        if device is None:
            device = packed.device if isinstance(packed, torch.Tensor) and packed.is_cuda else torch.device("cuda")
        canonical = _to_device_u8(packed, device)
        self.scales = _to_device_f16(scales, device)
        self.packed_v3 = ext().w4_repack(canonical, "v3") if "v3" in layouts else None
        self.packed_mma = ext().w4_repack(canonical, "mma") if "mma" in layouts else None
        self.packed = canonical if "canonical" in layouts else None

    @classmethod
    def from_float(cls, w, group=128, layouts=None):
        """Quantize a float weight [N, K] (on the GPU, bit-identical to quant.quantize_w4) and keep `layouts`."""
        packed, scales = quantize_w4_gpu(w, group)
        return cls(packed, scales, group, layouts)

    def __getstate__(self):
        """Without the launch arguments kept for this object's memory: a copy or an unpickled weight has its own."""
        return {name: v for name, v in self.__dict__.items() if name not in ("_launch", "_mma_launch")}

    def nbytes(self):
        """Bytes of one copy of the weight (packed values + scales), whatever layouts are kept."""
        return self.n * self.k // 2 + self.scales.numel() * 2

    def launch_args(self, version):
        """(packed pointer, scales pointer, device index) of the layout `version` reads, or None if that layout is
        not kept or not launchable; validated once per tensor object (replacing a layout tensor revalidates)."""
        if version == 5 or version == 6:   # the decode path: one attribute holds the mma copy's arguments
            hit = self.__dict__.get("_mma_launch")
            if hit is not None and hit[0] is self.packed_mma and hit[1] is self.scales:
                return hit[2]
        w, s = getattr(self, NEEDS[version]), self.scales
        cache = self.__dict__.setdefault("_launch", {})
        hit = cache.get(version)
        if hit is not None and hit[0] is w and hit[1] is s:
            return hit[2]
        args = None
        if (w is not None and w.is_cuda and s.is_cuda and w.device == s.device and w.dtype == torch.uint8
                and s.dtype == torch.float16 and w.is_contiguous() and s.is_contiguous() and w.dim() == 2
                and s.dim() == 2 and tuple(w.shape) == (self.n, self.k // 2) and self.group > 0
                and self.group % 32 == 0 and self.k % self.group == 0
                and tuple(s.shape) == (self.n, self.k // self.group)):
            args = (w.data_ptr(), s.data_ptr(), w.get_device())
        cache[version] = (w, s, args)
        if version == 5 or version == 6:
            self.__dict__["_mma_launch"] = (w, s, args)
        return args


def pick_rows(n, m):
    """Rows per warp the compatibility kernels (versions 1-4) use when rows_per_warp = 0 (csrc/w4_gemv.cu:424-427)."""
    return 4 if n >= 512 else 2 if m >= 4 else 1


# the layout each kernel version reads, and the most rows it takes
NEEDS = {1: "packed", 2: "packed", 3: "packed_v3", 4: "packed_v3", 5: "packed_mma", 6: "packed_mma"}
MAX_ROWS = {1: 8, 2: 8, 3: 8, 4: 8, 5: 64, 6: 8}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", None)
_F16 = torch.float16
_fast = None   # the _fastcall extension module, or False where it was not built (ctypes carries every call then)
_tc = None     # the _torchcall extension module (tensor checks in C++), or False where it was not built


def _current_stream(dev):
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


def _fastcall():
    global _fast
    if _fast is None:
        try:
            from . import _fastcall as fc
            ext()   # the library itself, loaded and checked by the ctypes binding (the extension links the same file)
            _fast = fc
        except ImportError:
            _fast = False
    return _fast


def _torchcall():
    global _tc
    if _tc is None:
        try:
            from . import _torchcall as tc
            ext()   # the library itself, loaded and checked by the ctypes binding (the extension links the same file)
            _tc = tc
        except ImportError:
            _tc = False
    return _tc


def _gemv_fast(x, wq, version, out, bias=None):
    """The common decode call with the weight's validated launch arguments cached: cheap checks on x, out and bias,
    one C call -- through the _torchcall extension (the checks in C++) when it was built, else the checks here and
    the _fastcall extension or ctypes. None when anything is unusual: the checked path below then handles it (and
    raises its errors)."""
    args = wq.launch_args(version)
    if args is None:
        return None
    tc = _tc if _tc is not None else _torchcall()
    if tc:
        return tc.gemv(x, args[0], args[1], args[2], wq.n, wq.k, wq.group, version, out, bias)
    if type(x) is not torch.Tensor or x.dtype is not _F16 or x.dim() != 2:
        return None
    w_ptr, s_ptr, dev = args
    m, kx = x.shape
    if (kx != wq.k or m == 0 or x.get_device() != dev or not x.is_contiguous()
            or (_raw_device() if _raw_device is not None else torch.cuda.current_device()) != dev):
        return None
    if bias is not None and (type(bias) is not torch.Tensor or bias.dtype is not _F16 or bias.dim() != 1
                             or bias.shape[0] != wq.n or bias.get_device() != dev or not bias.is_contiguous()):
        return None
    n = wq.n
    if out is None:
        y = torch.empty((m, n), dtype=_F16, device=x.device)
    elif (type(out) is torch.Tensor and out.dtype is _F16 and out.dim() == 2 and out.shape[0] == m
          and out.shape[1] == n and out.get_device() == dev and out.is_contiguous()):
        y = out
    else:
        return None
    fc = _fast if _fast is not None else _fastcall()
    st = _current_stream(dev)
    if fc:
        if bias is None:
            rc = fc.gemv(x.data_ptr(), w_ptr, s_ptr, y.data_ptr(), m, n, kx, wq.group, version, st)
        else:
            rc = fc.linear(x.data_ptr(), w_ptr, s_ptr, bias.data_ptr(), y.data_ptr(), m, n, kx, wq.group, version, st)
    else:
        lib = ext().lib
        if bias is not None:
            rc = lib.lb_w4_linear(x.data_ptr(), w_ptr, s_ptr, bias.data_ptr(), y.data_ptr(), m, n, kx, wq.group,
                                  version, st)
        elif version == 6:
            rc = lib.lb_w4_gemv(x.data_ptr(), w_ptr, s_ptr, y.data_ptr(), m, n, kx, wq.group, 6, 0, st)
        else:
            rc = lib.lb_w4_gemm_tc(x.data_ptr(), w_ptr, s_ptr, y.data_ptr(), m, n, kx, wq.group, 0, st)
    if rc:
        ext()._raise(rc)
    return y


def gemv(x, wq, version=4, rows_per_warp=0, out=None, bias=None):
    """x [M, K] fp16 -> [M, N] fp16. Versions 1-4 and 6: M <= 8; version 5: M <= 64 (tensor cores).
    Versions 5 and 6 read the same layout (packed_mma), so a model needs only that copy. `out`: an optional
    contiguous fp16 [M, N] tensor the result is written into (no allocation). `bias`: an optional fp16 [N] tensor
    added in the kernel's epilogue, with the roundings of adding it to the fp16 output afterwards (both are
    additions to the reference's signature)."""
    if (version == 5 or version == 6) and rows_per_warp == 0 and isinstance(wq, W4Weight):
        y = _gemv_fast(x, wq, version, out, bias)
        if y is not None:
            return y
    if version not in NEEDS:
        raise ValueError(f"version must be one of {sorted(NEEDS)}")
    if getattr(wq, NEEDS[version]) is None:
        raise ValueError(f"v{version} reads {NEEDS[version]}, which this W4Weight does not keep")
    if bias is not None:
        if rows_per_warp != 0:
            raise ValueError("rows_per_warp is chosen by the kernel when a bias is fused")
        return ext().w4_linear(x.contiguous(), getattr(wq, NEEDS[version]), wq.scales, wq.group, version, bias, out)
    if version == 5:
        return ext().w4_gemm_tc(x.contiguous(), wq.packed_mma, wq.scales, wq.group, rows_per_warp, out=out)
    w = wq.packed_mma if version == 6 else wq.packed_v3 if version >= 3 else wq.packed
    return ext().w4_gemv(x.contiguous(), w, wq.scales, wq.group, version, rows_per_warp, out=out)


_GEMV = gemv   # linear()'s shortcut applies only while ops.gemv is this function (tests may replace it)


def quantize_w4_gpu(w, group=128, clip_grid=None, rows_per_pass=2048):
    """Same format and, with clip_grid=None, the same bits as quant.quantize_w4, computed by the quantize kernel.
    clip_grid, e.g. (1.0, 0.95, ..., 0.75): per group, try scale = a * amax / 7 for each a and keep the first one
    with the smallest squared weight error. Returns (packed uint8 [N, K/2], scales fp16 [N, K/G]) on the GPU.
    Rows are converted and quantized `rows_per_pass` at a time, which bounds the fp32 staging copy
    (lowbit/ops.py:81-116)."""
    n, k = w.shape
    if group <= 0 or k % group or group % 32:
        raise ValueError(f"K={k} must be a multiple of the group size {group}, itself a multiple of 32")
    if clip_grid is not None and len(clip_grid) > 32:
        raise ValueError("clip_grid holds at most 32 factors")
    dev = w.device if isinstance(w, torch.Tensor) and w.is_cuda else torch.device("cuda")
    if not isinstance(w, torch.Tensor):
        w = torch.as_tensor(w)
    packed = torch.empty(n, k // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(n, k // group, dtype=torch.float16, device=dev)
    for r0 in range(0, n, rows_per_pass):
        part = w[r0:r0 + rows_per_pass].detach()
        if part.dtype not in (torch.float32, torch.float16):
            part = part.float()
        p, s = ext().w4_quantize(part.to(dev).contiguous(), group, clip_grid)
        packed[r0:r0 + rows_per_pass] = p
        scales[r0:r0 + rows_per_pass] = s
    return packed, scales


def dequantize_w4_gpu(packed, scales, group=128):
    """fp16 [N, K] from canonical packed weights on the GPU: (u - 8) * scale rounded once to fp16, the bits the
    reference's lowbit/ops.py:119-123 gives. Host arrays belong to quant.dequantize_w4."""
    if not (isinstance(packed, torch.Tensor) and packed.is_cuda):
        raise RuntimeError("dequantize_w4_gpu takes GPU tensors; use lowbit.quant.dequantize_w4 for host arrays")
    return ext().w4_dequant(packed.contiguous(), scales.contiguous(), group, layout="canonical")


def dequant(wq, layout=None):
    """fp16 W [N, K] from the canonical or the mma copy (None: canonical when kept). Both give the same bits."""
    if layout is None:
        layout = "canonical" if wq.packed is not None else "mma"
    if layout == "canonical" and wq.packed is not None:
        return ext().w4_dequant(wq.packed, wq.scales, wq.group)
    if layout == "mma" and wq.packed_mma is not None:
        return ext().w4_dequant(wq.packed_mma, wq.scales, wq.group, True)
    raise ValueError(f"cannot dequantize from the {layout} layout: not kept")


# ------------------------------------------------------------------------------------------ dispatch constants
#
# linear() picks, by row count and layer width: version 6 for up to AUTO_GEMV_ROWS rows, version 5 up to
# AUTO_V5_ROWS rows (AUTO_V5_WIDE_ROWS on layers with N >= AUTO_WIDE_N), dequantize + cuBLAS above. The values
# come from dispatch_b200.json (a B200 sweep). LOWBIT_DISPATCH=reference restores the reference's T4 values
# (lowbit/ops.py:142), under which the reference's own dispatch tests hold verbatim.

_REFERENCE_TABLE = {"AUTO_GEMV_ROWS": 1, "AUTO_V5_ROWS": 32, "AUTO_V5_WIDE_ROWS": 64, "AUTO_WIDE_N": 3072}
DISPATCH_TABLE_PATH = pathlib.Path(__file__).resolve().parent / "dispatch_b200.json"


def _load_dispatch():
    if os.environ.get("LOWBIT_DISPATCH", "") == "reference":
        return dict(_REFERENCE_TABLE, source="reference T4 constants (lowbit/ops.py:142)")
    table = json.loads(DISPATCH_TABLE_PATH.read_text())
    return table


DISPATCH = _load_dispatch()
AUTO_GEMV_ROWS, AUTO_V5_ROWS, AUTO_V5_WIDE_ROWS, AUTO_WIDE_N = (
    int(DISPATCH[k]) for k in ("AUTO_GEMV_ROWS", "AUTO_V5_ROWS", "AUTO_V5_WIDE_ROWS", "AUTO_WIDE_N"))


def gemm_chunked(x, wq, chunk=64):
    """Many rows through version 5 in 64-row slices (no fp16 weight copy is written)."""
    return torch.cat([gemv(x[i:i + chunk], wq, 5) for i in range(0, x.shape[0], chunk)])


def auto_version(m, wq):
    """The kernel linear() uses for m rows, or None for dequantize + cuBLAS. Weights without the mma layout use
    version 4 / 2 up to 8 rows (lowbit/ops.py:151-160)."""
    if wq.packed_mma is not None:
        if m <= AUTO_GEMV_ROWS:
            return 6
        return 5 if m <= (AUTO_V5_WIDE_ROWS if wq.n >= AUTO_WIDE_N else AUTO_V5_ROWS) else None
    if m <= 8:
        return 4 if wq.packed_v3 is not None else 2 if wq.packed is not None else None
    return None


def linear(x, wq, max_gemv_rows=8, version=0, out=None, bias=None):
    """Decode (few rows): an INT4 kernel; prefill (many rows): dequantize, then cuBLAS fp16 GEMM. version 0 =
    auto_version; a fixed version runs up to min(max_gemv_rows, its row limit) rows (version 5: 64), and
    dequantize + cuBLAS above that (lowbit/ops.py:163-178). Additions to the reference's signature: `out`, an
    optional contiguous fp16 [M, N] tensor that receives the result, and `bias`, an optional fp16 [N] tensor added
    to the result (in the INT4 kernels' epilogue; after the cuBLAS product on the prefill path) with the roundings
    of adding it to the fp16 output."""
    m = x.shape[0]
    if version == 0 and m and type(wq) is W4Weight and wq.packed_mma is not None and gemv is _GEMV:
        # the decode call: the rule of auto_version inline, straight to the cached launch (anything unusual falls
        # through to the general path below)
        v = 6 if m <= AUTO_GEMV_ROWS else 5 if m <= (AUTO_V5_WIDE_ROWS if wq.n >= AUTO_WIDE_N else AUTO_V5_ROWS) else 0
        if v:
            y = _gemv_fast(x, wq, v, out, bias)
            if y is not None:
                return y
    if m == 0:
        return x.new_empty(0, wq.n) if out is None else out
    if version == 0:
        v = auto_version(m, wq)
    elif version in MAX_ROWS:
        v = version if m <= (MAX_ROWS[5] if version == 5 else min(max_gemv_rows, MAX_ROWS[version])) else None
    else:
        raise ValueError(f"version must be 0 (auto) or one of {sorted(MAX_ROWS)}")
    if v is not None:
        if bias is not None:
            return gemv(x, wq, v, out=out, bias=bias)
        return gemv(x, wq, v) if out is None else gemv(x, wq, v, out=out)
    y = torch.nn.functional.linear(x, dequant(wq, "mma" if wq.packed_mma is not None else "canonical"))
    if bias is not None:
        y = y + bias
    if out is None:
        return y
    if out.shape != y.shape or out.dtype != y.dtype:
        raise RuntimeError(f"out must be a float16 {tuple(y.shape)} tensor")
    return out.copy_(y)


# ------------------------------------------------------------------------------------------ 8-bit integer products
#
# W8A8: weights in 8-bit integers with one fp32 scale per output channel, activations quantized per token on the way
# into the product, sums exact in int32 (lb_w8_linear). For prompts: twice the tensor-core rate of the dequantize +
# fp16 path, and half its weight bytes. No counterpart in the reference.

def quantize_w8_gpu(w):
    """(int8 [N, K], scales fp32 [N]) of a float weight [N, K] (fp16, bf16 or fp32, on the GPU): per output channel
    scale = max|w| / 127 and q = rint(w * (127 / max|w|)), half to even. The same rule per token is what linear_w8
    applies to its activations."""
    if not (isinstance(w, torch.Tensor) and w.is_cuda):
        raise RuntimeError("quantize_w8_gpu takes GPU tensors")
    if w.dim() != 2 or w.dtype not in DTYPE_IDS:
        raise RuntimeError("w must be a float16, bfloat16 or float32 [N, K] tensor")
    n, k = w.shape
    if w.stride(1) != 1 or w.stride(0) < k:
        w = w.contiguous()
    q = torch.empty(n, -(-k // 16) * 16, dtype=torch.int8, device=w.device)
    scales = torch.empty(n, dtype=torch.float32, device=w.device)
    e = ext()
    if n and k:
        with _Device(w.device):
            rc = e.lib.lb_w8_quantize_rows(w.data_ptr(), DTYPE_IDS[w.dtype], n, k, w.stride(0) if n > 1 else k,
                                           q.data_ptr(), q.shape[1], scales.data_ptr(),
                                           torch.cuda.current_stream().cuda_stream)
        if rc:
            e._raise(rc)
    return q[:, :k], scales


class W8Weight:
    """One linear layer's weight in 8-bit integers on the GPU: q int8 [N, K], scales fp32 [N] (W = q * scale). A q
    whose K and row stride are multiples of 16 is kept without a copy, any other is laid out once with zeros behind K."""

    def __init__(self, q, scales):
        if not (isinstance(q, torch.Tensor) and isinstance(scales, torch.Tensor) and q.is_cuda):
            raise RuntimeError("W8Weight takes GPU tensors")
        if q.dtype != torch.int8 or q.dim() != 2 or not q.numel():
            raise RuntimeError("q must be an int8 [N, K] tensor")
        self.n, self.k = q.shape   # no device pointer is kept: a copy or an unpickled weight has its own memory
        if scales.dtype != torch.float32 or scales.shape != (self.n,) or scales.device != q.device:
            raise RuntimeError(f"scales must be a float32 [{self.n}] tensor on {q.device}")
        if self.k > 131072:
            raise ValueError(f"K={self.k}: at most 131072, so that the int32 sums are exact")
        if (self.k % 16 == 0 and q.stride(1) == 1 and q.stride(0) % 16 == 0 and q.stride(0) >= self.k
                and q.data_ptr() % 16 == 0):
            self._q = q
        else:
            pad = torch.zeros(self.n, -(-self.k // 16) * 16, dtype=torch.int8, device=q.device)
            pad[:, :self.k] = q
            self._q = pad[:, :self.k]
        self._scales = scales.contiguous()

    @property
    def q(self):
        return self._q

    @property
    def scales(self):
        return self._scales

    @classmethod
    def from_float(cls, w):
        return cls(*quantize_w8_gpu(w))

    def nbytes(self):
        return self.n * self.k + 4 * self.n


def linear_w8(x, w8, bias=None, out=None):
    """x [M, K] fp16 or bf16 (rows any stride apart) -> [M, N] of the same type: each row quantized to 8-bit integers
    with its own scale, the product with w8 (W8Weight) exact in int32, then scaled, `bias` ([N], x's type) added and
    rounded once. `out`: an optional contiguous [M, N] tensor that receives the result. A serving operator: the result
    carries no autograd graph."""
    tc = _tc if _tc is not None else _torchcall()
    if tc:
        y = tc.linear_w8(x, w8._q, w8._scales, out, bias)
        if y is not None:
            return y
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.device == w8.q.device):
        raise RuntimeError(f"x must be on the weight's GPU, {w8.q.device}")
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2 or x.shape[1] != w8.k:
        raise RuntimeError(f"x must be a float16 or bfloat16 [M, {w8.k}] tensor")
    m = x.shape[0]
    if bias is not None and (not bias.is_cuda or bias.device != x.device or bias.dtype != x.dtype
                             or bias.shape != (w8.n,) or not bias.is_contiguous()):
        raise RuntimeError(f"bias must be a contiguous {x.dtype} [{w8.n}] tensor on {x.device}")
    if out is None:
        out = torch.empty(m, w8.n, dtype=x.dtype, device=x.device)
    elif out.shape != (m, w8.n) or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise RuntimeError(f"out must be a contiguous {x.dtype} [{m}, {w8.n}] tensor on {x.device}")
    if m == 0:
        return out
    if x.stride(1) != 1 or (m > 1 and x.stride(0) < w8.k):
        x = x.contiguous()
    e = ext()
    n, k, ldw = w8.n, w8.k, w8.q.stride(0) if w8.n > 1 else -(-w8.k // 16) * 16
    with _Device(x.device):
        need = e.lib.lb_w8_workspace(m, n, k)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        rc = e.lib.lb_w8_linear(x.data_ptr(), DTYPE_IDS[x.dtype], x.stride(0) if m > 1 else k, w8.q.data_ptr(), ldw,
                                w8.scales.data_ptr(),
                                None if bias is None else bias.data_ptr(), out.data_ptr(), m, n, k,
                                ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream)
    if rc:
        e._raise(rc)
    return out


# ------------------------------------------------------------------------------------------ 8-bit floating point
#
# Weights in e4m3 with one fp32 scale per 128 x 128 block, activations quantized per token and 128 values on the way into
# the product (lb_f8_linear): the format of block-scaled 8-bit checkpoints. No counterpart in the reference.

F8_BLOCK = 128


def _f8_blocks(n):
    return -(-n // F8_BLOCK)


def quantize_f8_gpu(w):
    """(float8_e4m3fn [N, K], scales fp32 [ceil(N / 128), ceil(K / 128)]) of a float weight [N, K] (fp16, bf16 or fp32, on the
    GPU): per 128 x 128 block a = max(max|w|, 2^-100), scale = a / 448 and q = w * (448 / a) rounded to nearest even. The
    same rule per token and 128 values is what linear_f8 applies to its activations."""
    if not (isinstance(w, torch.Tensor) and w.is_cuda):
        raise RuntimeError("quantize_f8_gpu takes GPU tensors")
    if w.dim() != 2 or w.dtype not in DTYPE_IDS:
        raise RuntimeError("w must be a float16, bfloat16 or float32 [N, K] tensor")
    n, k = w.shape
    if w.stride(1) != 1 or w.stride(0) < k:
        w = w.contiguous()
    q = torch.empty(n, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=w.device)
    scales = torch.empty(_f8_blocks(n), _f8_blocks(k), dtype=torch.float32, device=w.device)
    e = ext()
    if n and k:
        with _Device(w.device):
            rc = e.lib.lb_f8_quantize_weight(w.data_ptr(), DTYPE_IDS[w.dtype], n, k, w.stride(0) if n > 1 else k, q.data_ptr(),
                                             q.shape[1], scales.data_ptr(), torch.cuda.current_stream().cuda_stream)
        if rc:
            e._raise(rc)
    return q[:, :k], scales


class F8Weight:
    """One linear layer's weight in 8-bit floating point on the GPU: q float8_e4m3fn [N, K], scales fp32 [ceil(N / 128),
    ceil(K / 128)] (W = q * its block's scale). A q whose K and row stride are multiples of 16 is kept without a copy, any other
    is laid out once with zeros behind K."""

    def __init__(self, q, scales):
        if not (isinstance(q, torch.Tensor) and isinstance(scales, torch.Tensor) and q.is_cuda):
            raise RuntimeError("F8Weight takes GPU tensors")
        if q.dtype != torch.float8_e4m3fn or q.dim() != 2 or not q.numel():
            raise RuntimeError("q must be a float8_e4m3fn [N, K] tensor")
        self.n, self.k = q.shape   # no device pointer is kept: a copy or an unpickled weight has its own memory
        blocks = (_f8_blocks(self.n), _f8_blocks(self.k))
        if scales.dtype != torch.float32 or scales.shape != blocks or scales.device != q.device:
            raise RuntimeError(f"scales must be a float32 {list(blocks)} tensor on {q.device}")
        if self.k > 131072:
            raise ValueError(f"K={self.k}: at most 131072")
        if (self.k % 16 == 0 and q.stride(1) == 1 and q.stride(0) % 16 == 0 and q.stride(0) >= self.k
                and q.data_ptr() % 16 == 0):
            self._q = q.view(torch.uint8)   # as bytes: torch does not pickle tensors of this type
        else:
            pad = torch.zeros(self.n, -(-self.k // 16) * 16, dtype=torch.uint8, device=q.device)
            pad[:, :self.k] = q.view(torch.uint8)
            self._q = pad[:, :self.k]
        self._scales = scales.contiguous()

    @property
    def q(self):
        return self._q.view(torch.float8_e4m3fn)

    @property
    def scales(self):
        return self._scales

    @classmethod
    def from_float(cls, w):
        return cls(*quantize_f8_gpu(w))

    def nbytes(self):
        return self.n * self.k + 4 * self._scales.numel()


def linear_f8(x, f8, bias=None, out=None):
    """x [M, K] fp16 or bf16 (rows any stride apart) -> [M, N] of the same type: each row quantized to e4m3 with a scale per 128
    values, the product with f8 (F8Weight) summed in fp32, each block times its two scales, `bias` ([N], x's type) added and
    rounded once. `out`: an optional contiguous [M, N] tensor that receives the result, not over x. A serving operator:
    the result carries no autograd graph."""
    tc = _tc if _tc is not None else _torchcall()
    if tc:
        y = tc.linear_f8(x, f8._q, f8._scales, out, bias)
        if y is not None:
            return y
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.device == f8._q.device):
        raise RuntimeError(f"x must be on the weight's GPU, {f8._q.device}")
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2 or x.shape[1] != f8.k:
        raise RuntimeError(f"x must be a float16 or bfloat16 [M, {f8.k}] tensor")
    m = x.shape[0]
    if bias is not None and (not bias.is_cuda or bias.device != x.device or bias.dtype != x.dtype
                             or bias.shape != (f8.n,) or not bias.is_contiguous()):
        raise RuntimeError(f"bias must be a contiguous {x.dtype} [{f8.n}] tensor on {x.device}")
    if out is None:
        out = torch.empty(m, f8.n, dtype=x.dtype, device=x.device)
    elif out.shape != (m, f8.n) or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise RuntimeError(f"out must be a contiguous {x.dtype} [{m}, {f8.n}] tensor on {x.device}")
    if m == 0:
        return out
    if x.stride(1) != 1 or (m > 1 and x.stride(0) < f8.k):
        x = x.contiguous()
    e = ext()
    n, k, ldw = f8.n, f8.k, f8._q.stride(0) if f8.n > 1 else -(-f8.k // 16) * 16
    with _Device(x.device):
        need = e.lib.lb_f8_workspace(m, n, k)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        rc = e.lib.lb_f8_linear(x.data_ptr(), DTYPE_IDS[x.dtype], x.stride(0) if m > 1 else k, f8._q.data_ptr(), ldw,
                                f8._scales.data_ptr(),
                                None if bias is None else bias.data_ptr(), out.data_ptr(), m, n, k,
                                ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream)
    if rc:
        e._raise(rc)
    return out
