"""BF16 skinny projections on B200.

Drop-in for engine/kernels/linear.py:489-523 ``linear(x, weight, split_ok)``: all products
accumulate in FP32 and round once to BF16. Decode-sized inputs (<= MAX_ROWS rows, aligned
K/N) run the TMA + mma.sync kernel fb_linear over (N/128 tiles) x (K splits); with
``split_ok`` a split-K result comes back as a ``Split`` of FP32 partials for a consumer kernel
to sum (merged.py), otherwise the split CTAs of each tile form a thread-block cluster that sums
the tile's partials in split order and writes BF16 (same launch). Larger row counts (prefill)
stay on cuBLAS through ``F.linear``, exactly as the reference routes them (linear.py:492).

``keep_native`` is the reference's hook for leaving a shape on cuBLAS without tuning it
(linear.py:484-486); the B200 kernels choose their launch shape by a fixed rule (no timed
search), so it only records the request.

``linear``, ``swiglu_linear`` and ``project`` also take 4-bit weights (kernels.quant.Weight4):
fb_linear_w4 for every MAX_ROWS rows up to MAX_ROWS4, one launch each whose result is finished (never a
``Split``); more rows go to cuBLAS on the weights expanded to BF16 for the call. The reference has no such form.
"""

import torch
from torch.nn import functional as F

from kernels import _native
from kernels._native import check, launch, lib, ptr, stream
from kernels.merged import Split
from kernels.quant import Weight4

#: Rows the skinny kernel takes (x is staged as 16/32/64-row slabs).
MAX_ROWS = 64
#: Rows that 4-bit weights take in launches of MAX_ROWS. 65 and 128 rows in two launches against expanded weights
#: and cuBLAS, us: [4096, 4096] 16.0 and 18.5 against 22.8 and 23.0, [4096, 12288] 27 and 32 against 66, [24576, 4096] 57
#: and 76 against 123 and 125, but [4096, 1024] 11.3 and 12.8 against 8.8. Three launches of 192 rows of
#: [4096, 4096]: 26.8 against 21.9.
MAX_ROWS4 = 2 * MAX_ROWS
BF16_OUT, FP32_OUT, SWIGLU_OUT, SPLITS_OUT = 0, 1, 2, 3
_SPLITS = {}


def splits_for(rows, n, k, device, finished=False):
    """fb_linear_splits' choice, or fb_linear_finished_splits' for finished-tile epilogues."""
    key = (device, rows, n, k, finished)
    if key not in _SPLITS:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("projection selection must finish during eager warmup")
        choose = lib.fb_linear_finished_splits if finished else lib.fb_linear_splits
        _SPLITS[key] = int(choose(rows, n, k))
    return _SPLITS[key]


def keep_native(rows, weight):
    """engine/kernels/linear.py:484-486: leave ``rows`` x ``weight`` on cuBLAS without spending
    tuning time on it. The B200 projection has no timed search to skip, and the reference calls
    this only for row counts above MAX_ROWS (its verify blocks), which ``linear`` already routes
    to cuBLAS; the shape is recorded so ``linear`` keeps it there whatever its row count. Products
    with 4-bit weights keep their own rule: cuBLAS would need the weights expanded."""
    _NATIVE.add((weight.device, rows, weight.shape[0], weight.shape[1]))


_NATIVE = set()


def supported(rows, weight):
    n, k = weight.shape
    return 0 < rows <= MAX_ROWS and k % 8 == 0 and n % 8 == 0 and weight.dtype == torch.bfloat16


def project(flat, weight, epilogue=BF16_OUT, splits=None):
    """fb_linear on [M,K] x [N,K]: BF16 [M,N], FP32 [M,N], SwiGLU BF16 [M,N/2] or FP32 split
    partials [S,M,N] (4-bit weights: S is 1)."""
    if isinstance(weight, Weight4):
        return _project4(flat, weight, epilogue)
    m, k = flat.shape
    n = weight.shape[0]
    if splits is None:
        splits = splits_for(m, n, k, flat.device, finished=epilogue != SPLITS_OUT)
    if epilogue == SWIGLU_OUT:
        out = torch.empty((m, n // 2), device=flat.device, dtype=torch.bfloat16)
    elif epilogue == SPLITS_OUT:
        out = torch.empty((splits, m, n), device=flat.device, dtype=torch.float32)
    else:
        out = torch.empty((m, n), device=flat.device, dtype=torch.float32 if epilogue == FP32_OUT else torch.bfloat16)
    check(lib.fb_linear(ptr(flat), ptr(weight), ptr(out), m, n, k, epilogue, splits, stream()), "fb_linear")
    return out


def _launch4(x, weight, out, rows, epilogue):
    """fb_linear_w4 on contiguous x of ``rows`` rows, MAX_ROWS of them at a time."""
    device = weight.device
    if x.device != device:
        raise ValueError(f"4-bit weights on {device} take inputs of that device, not {x.device}")
    if x.data_ptr() % 16:
        x = x.clone()
    source, target, packed = x.data_ptr(), out.data_ptr(), weight.packed.data_ptr()
    n, k, group = weight.n, weight.k, weight.group
    launch("fb_linear_w4", device, source, packed, target, min(rows, MAX_ROWS), n, k, group, epilogue)
    for row in range(MAX_ROWS, rows, MAX_ROWS):
        launch("fb_linear_w4", device, source + row * k * 2, packed, target + row * (out.nbytes // rows),
               min(rows - row, MAX_ROWS), n, k, group, epilogue)
    return out


def _refuse4(x, weight):
    raise ValueError(f"4-bit weights {tuple(weight.shape)} take 1 to {MAX_ROWS4} BF16 rows of their width, not "
                     f"{x.dtype} {tuple(x.shape)}")


def _project4(flat, weight, epilogue):
    """fb_linear_w4 on [M,K]: the outputs of ``project``."""
    m, n = flat.shape[0], weight.n
    if flat.shape[1] != weight.k or flat.dtype != torch.bfloat16 or not 0 < m <= MAX_ROWS4:
        _refuse4(flat, weight)
    if epilogue == SWIGLU_OUT:
        if n % 128:
            raise ValueError(f"SwiGLU weights are 64-row gate/up blocks: {n} rows are not a multiple of 128")
        out = flat.new_empty(m, n // 2)
    elif epilogue == BF16_OUT:
        out = flat.new_empty(m, n)
    else:
        out = flat.new_empty((1, m, n) if epilogue == SPLITS_OUT else (m, n), dtype=torch.float32)
    return _launch4(flat.contiguous(), weight, out, m, FP32_OUT if epilogue == SPLITS_OUT else epilogue)


def _linear4(x, weight):
    shape, k = x.shape, weight.k
    if shape[-1] != k or x.dtype != torch.bfloat16:
        _refuse4(x, weight)
    rows = x.numel() // k
    if rows > MAX_ROWS4:
        _native.require_device(weight.device, x)
        return F.linear(x, weight.dequantized())
    out = x.new_empty(*shape[:-1], weight.n)
    return _launch4(x if x.is_contiguous() else x.contiguous(), weight, out, rows, BF16_OUT) if rows else out


def linear(x, weight, split_ok=False):
    """x @ weight.T in BF16. With ``split_ok`` the result may be a ``Split`` for a consumer kernel.
    ``weight``: a BF16 [N, K] tensor or a ``Weight4``."""
    if isinstance(weight, Weight4):
        return _linear4(x, weight)
    rows = x.numel() // x.shape[-1]
    if x.dtype != torch.bfloat16 or not weight.is_contiguous() or not supported(rows, weight):
        return F.linear(x, weight)
    if _NATIVE and (weight.device, rows, weight.shape[0], weight.shape[1]) in _NATIVE:
        return F.linear(x, weight)
    _native.require_cuda(x, weight)
    flat = x.reshape(rows, x.shape[-1]).contiguous()
    n, k = weight.shape
    splits = splits_for(rows, n, k, x.device)
    if split_ok and splits > 1:
        return Split(project(flat, weight, SPLITS_OUT, splits), (*x.shape[:-1], n))
    return project(flat, weight, BF16_OUT, splits_for(rows, n, k, x.device, finished=True)).reshape(
        *x.shape[:-1], n)


def swiglu_linear(x, gate_up_blocked):
    """SwiGLU(x @ W^T), W's rows being [gate; up] interleaved in 64-row blocks: bf16(bf16(silu(
    gate)) * up) per feature, the reference's projection + swiglu arithmetic. At one K split the
    projection's epilogue applies SwiGLU (one launch). With K splits the projection writes
    split partials that fb_swiglu_blocked sums and activates (measured faster inside the decode
    step than summing the splits in the projection's own launch). The same bits either way."""
    rows = x.numel() // x.shape[-1]
    flat = x.reshape(rows, x.shape[-1]).contiguous()
    n, k = gate_up_blocked.shape
    if isinstance(gate_up_blocked, Weight4):  # finished in the projection's launch
        return _project4(flat, gate_up_blocked, SWIGLU_OUT).view(*x.shape[:-1], n // 2)
    splits = splits_for(rows, n, k, x.device)
    if splits == 1:
        return project(flat, gate_up_blocked, SWIGLU_OUT, splits).reshape(*x.shape[:-1], n // 2)
    partials = project(flat, gate_up_blocked, SPLITS_OUT, splits)
    out = torch.empty((rows, n // 2), device=x.device, dtype=torch.bfloat16)
    check(lib.fb_swiglu_blocked(ptr(partials), splits, ptr(out), rows, n // 2, stream()), "fb_swiglu_blocked")
    return out.reshape(*x.shape[:-1], n // 2)
