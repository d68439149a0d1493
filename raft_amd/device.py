"""Pass torch device tensors through the C ABI (device memory and streams only).

torch provides allocation, the current HIP stream and events; every reduction
is computed by libraft_amd.so.  A missing library or a non-OK status raises.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _capi as api


class RmiError(RuntimeError):
    def __init__(self, code: int, where: str):
        super().__init__(f"{where}: {api.status_string(code)} (status {code})")
        self.code = code


def current_stream_ptr() -> int:
    return torch.cuda.current_stream().cuda_stream


def workspace_for(desc: api.ReduceDesc, device="cuda") -> torch.Tensor | None:
    n = api.load().rmi_reduce_workspace_bytes(C.byref(desc))
    if n == 0:
        return None
    return torch.empty(n, dtype=torch.uint8, device=device)


def reduce(desc: api.ReduceDesc, inp: torch.Tensor, out: torch.Tensor,
           workspace: torch.Tensor | None = None, *, in_ptr: int | None = None,
           out_ptr: int | None = None) -> None:
    """Run rmi_reduce on the current torch stream.  `inp` / `out` are device tensors
    whose storage is interpreted according to the descriptor's dtypes."""
    lib = api.load()
    if workspace is None:
        workspace = workspace_for(desc, inp.device if inp is not None else out.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    ip = in_ptr if in_ptr is not None else (inp.data_ptr() if inp is not None else None)
    op = out_ptr if out_ptr is not None else out.data_ptr()
    rc = lib.rmi_reduce(C.byref(desc), ip, op, ws_ptr, ws_bytes, current_stream_ptr())
    if rc != api.OK:
        raise RmiError(rc, "rmi_reduce")


def map_reduce(desc: api.ReduceDesc, length: int, inp: torch.Tensor, out: torch.Tensor) -> None:
    lib = api.load()
    n = lib.rmi_map_reduce_workspace_bytes(C.byref(desc), length)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=inp.device)
    rc = lib.rmi_map_reduce(C.byref(desc), length, inp.data_ptr(), out.data_ptr(),
                            ws.data_ptr(), n, current_stream_ptr())
    if rc != api.OK:
        raise RmiError(rc, "rmi_map_reduce")


def meanvar(dtype: int, layout: int, n_rows: int, n_cols: int, sample: bool,
            data: torch.Tensor, mean: torch.Tensor, var: torch.Tensor) -> None:
    """Run rmi_meanvar on the current torch stream."""
    lib = api.load()
    n = lib.rmi_meanvar_workspace_bytes(dtype, layout, n_rows, n_cols)
    ws = torch.empty(n, dtype=torch.uint8, device=data.device) if n else None
    rc = lib.rmi_meanvar(dtype, layout, n_rows, n_cols, 1 if sample else 0, data.data_ptr(),
                         mean.data_ptr(), var.data_ptr(), ws.data_ptr() if n else None, n,
                         current_stream_ptr())
    if rc != api.OK:
        raise RmiError(rc, "rmi_meanvar")


def cov(dtype: int, layout: int, n_rows: int, n_cols: int, sample: bool, data: torch.Tensor,
        mu: torch.Tensor | None, covar: torch.Tensor, *, center: bool = False) -> None:
    """Run rmi_cov on the current torch stream; with `center` the call leaves x - mu in `data`."""
    lib = api.load()
    n = lib.rmi_cov_workspace_bytes(dtype, layout, n_rows, n_cols)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=covar.device)
    rc = lib.rmi_cov(dtype, layout, n_rows, n_cols, 1 if sample else 0,
                     api.COV_CENTER_DATA if center else 0,
                     data.data_ptr() if data is not None else None,
                     mu.data_ptr() if mu is not None else None, covar.data_ptr(), ws.data_ptr(), n,
                     current_stream_ptr())
    if rc != api.OK:
        raise RmiError(rc, "rmi_cov")


# ---- rows of logits -------------------------------------------------------------------------------

_LOGITS_DTYPE = {torch.float16: api.F16, torch.bfloat16: api.BF16, torch.float32: api.F32}
# the address of a device's current stream, without a Stream object around it where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _dtype_of(t: torch.Tensor, what: str) -> int:
    d = _LOGITS_DTYPE.get(t.dtype)
    if d is None:
        raise ValueError(f"{what}: float16, bfloat16 or float32 is wanted, got {t.dtype}")
    return d


def _logits(x: torch.Tensor, what: str = "logits") -> tuple[int, int, int, int]:
    """dtype, rows, columns and row stride of a matrix whose rows are contiguous."""
    d = _dtype_of(x, what)
    if x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"{what}: a matrix on the GPU is wanted")
    n_rows, n_cols = x.shape
    ld, step = x.stride()
    if step != 1 and n_cols > 1:
        raise ValueError(f"{what}: the elements of a row have to be contiguous")
    if ld < n_cols:
        if n_rows > 1:
            raise ValueError(f"{what}: rows overlap")
        ld = n_cols
    return d, n_rows, n_cols, ld


def _ptr(t: torch.Tensor | None, shape: tuple, dtype, device: int, what: str) -> int | None:
    """Address of a contiguous tensor of that shape and type on that GPU; None stays None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} tensor of shape {tuple(shape)} on GPU {device} is wanted, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _call(name: str, device: int, *args) -> None:
    """The library's call with that device current, on its current stream."""
    fn = getattr(api.load(), name)
    if device == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc != api.OK:
        raise RmiError(rc, name)


def top_k(x: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, lse: torch.Tensor | None = None, *,
          temperature: float = 1.0) -> None:
    """Run rmi_top_k on the current torch stream: the k = values.shape[1] elements of every row of
    `x` that rank first (int32 `indices`), and log(sum(exp(x / temperature))) of every row."""
    d, n_rows, n_cols, ld = _logits(x)
    device, shape = x.get_device(), (n_rows, values.shape[-1])
    _call("rmi_top_k", device, d, n_rows, n_cols, ld, shape[1], temperature, x.data_ptr(),
          _ptr(values, shape, x.dtype, device, "values"), _ptr(indices, shape, torch.int32, device, "indices"),
          _ptr(lse, (n_rows,), torch.float32, device, "lse"))


def _teacher(n_rows: int, device: int, t_values, t_indices, teacher_lse) -> tuple:
    shape = (n_rows, t_values.shape[-1])
    return (_ptr(t_values, shape, t_values.dtype, device, "t_values"),
            _ptr(t_indices, shape, torch.int32, device, "t_indices"),
            _ptr(teacher_lse, (n_rows,), torch.float32, device, "teacher_lse"))


def _grad(x: torch.Tensor, grad: torch.Tensor | None) -> tuple[int | None, int]:
    if grad is None:
        return None, 0
    if grad.dtype is not x.dtype or grad.shape != x.shape or grad.get_device() != x.get_device():
        raise ValueError("grad: the type, shape and device of the logits are wanted")
    return grad.data_ptr(), _logits(grad, "grad")[3]


def distill_loss(x: torch.Tensor, t_values: torch.Tensor, t_indices: torch.Tensor, loss: torch.Tensor,
                 stats: torch.Tensor | None = None, grad: torch.Tensor | None = None, *, temperature: float = 1.0,
                 scale: float = 1.0, teacher_lse: torch.Tensor | None = None,
                 row_grad: torch.Tensor | None = None) -> None:
    """Run rmi_distill_loss on the current torch stream: the loss of every row of student logits
    against a teacher's stored best logits; `stats` ([rows, 2]) for distill_grad, or the gradient at
    once in `grad`, which may be `x`.  Autograd records nothing here: logits that came out of a model
    take the gradient on by `x.backward(grad)`."""
    d, n_rows, n_cols, ld = _logits(x)
    device = x.get_device()
    _call("rmi_distill_loss", device, d, _dtype_of(t_values, "t_values"), n_rows, n_cols, ld, t_values.shape[-1],
          temperature, scale, x.data_ptr(), *_teacher(n_rows, device, t_values, t_indices, teacher_lse),
          _ptr(loss, (n_rows,), torch.float32, device, "loss"), _ptr(stats, (n_rows, 2), torch.float32, device, "stats"),
          _ptr(row_grad, (n_rows,), torch.float32, device, "row_grad"), *_grad(x, grad))


def distill_grad(x: torch.Tensor, t_values: torch.Tensor, t_indices: torch.Tensor, stats: torch.Tensor,
                 grad: torch.Tensor, *, temperature: float = 1.0, scale: float = 1.0,
                 teacher_lse: torch.Tensor | None = None, row_grad: torch.Tensor | None = None) -> None:
    """Run rmi_distill_grad on the current torch stream: the gradient of an earlier distill_loss from
    its `stats`, for the gradient `row_grad` of every row's loss (None: ones); for use in a backward
    pass of the caller's own, as autograd records nothing of either call."""
    d, n_rows, n_cols, ld = _logits(x)
    device = x.get_device()
    _call("rmi_distill_grad", device, d, _dtype_of(t_values, "t_values"), n_rows, n_cols, ld, t_values.shape[-1],
          temperature, scale, x.data_ptr(), *_teacher(n_rows, device, t_values, t_indices, teacher_lse),
          _ptr(stats, (n_rows, 2), torch.float32, device, "stats"),
          _ptr(row_grad, (n_rows,), torch.float32, device, "row_grad"), *_grad(x, grad))


def sample(x: torch.Tensor, u: torch.Tensor, token: torch.Tensor, logprob: torch.Tensor | None = None, *,
           temperature: torch.Tensor | None = None, top_k: torch.Tensor | None = None,
           top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           allowed: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> None:
    """Run rmi_sample on the current torch stream: one int32 `token` of every row of `x` for the
    random numbers `u`, with one setting per row (`top_k` int32, the others float32), and among the
    tokens whose bit is set in `allowed` ([rows, ceil(vocabulary / 32)] int32 or uint32 words).
    `workspace`: bytes that a caller keeps for it (rmi_sample_workspace_bytes), else allocated here."""
    d, n_rows, n_cols, ld = _logits(x)
    device, rows, f32 = x.get_device(), (n_rows,), torch.float32
    ap, lda = None, 0
    if allowed is not None:
        words = (n_cols + 31) // 32
        if (allowed.dtype not in (torch.int32, torch.uint32) or allowed.shape != (n_rows, words)
                or (allowed.stride(1) != 1 and words > 1) or (n_rows > 1 and allowed.stride(0) < words)
                or allowed.get_device() != device):
            raise ValueError(f"allowed: [{n_rows}, {words}] 32-bit words on GPU {device} are wanted")
        ap, lda = allowed.data_ptr(), max(allowed.stride(0), words)
    if workspace is None:
        n = api.load().rmi_sample_workspace_bytes(d, n_rows, n_cols)
        workspace = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
    elif workspace.get_device() != device:
        raise ValueError(f"workspace: memory on GPU {device} is wanted")
    wp, wn = (workspace.data_ptr(), workspace.nbytes) if workspace is not None else (None, 0)
    _call("rmi_sample", device, d, n_rows, n_cols, ld, x.data_ptr(), ap, lda,
          _ptr(temperature, rows, f32, device, "temperature"), _ptr(top_k, rows, torch.int32, device, "top_k"),
          _ptr(top_p, rows, f32, device, "top_p"), _ptr(min_p, rows, f32, device, "min_p"), _ptr(u, rows, f32, device, "u"),
          _ptr(token, rows, torch.int32, device, "token"), _ptr(logprob, rows, f32, device, "logprob"), wp, wn)
