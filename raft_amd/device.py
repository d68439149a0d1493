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
    (n_rows, n_cols), (ld, step) = x.shape, x.stride()
    if step != 1 and n_cols > 1:
        raise ValueError(f"{what}: the elements of a row have to be contiguous")
    if n_rows > 1 and ld < n_cols:
        raise ValueError(f"{what}: rows overlap")
    return d, n_rows, n_cols, max(ld, n_cols)


def _ptr(t: torch.Tensor | None, shape: tuple, dtype, like: torch.Tensor, what: str) -> int | None:
    """Address of a contiguous tensor of that shape and type beside `like`; None stays None."""
    if t is None:
        return None
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{what}: a contiguous {dtype} tensor of shape {tuple(shape)} on {like.device} is wanted, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _workspace(given: torch.Tensor | None, n: int, like: torch.Tensor) -> tuple[torch.Tensor | None, int | None, int]:
    if given is None and n > 0:
        given = torch.empty(n, dtype=torch.uint8, device=like.device)
    if given is None:
        return None, None, 0
    if given.device != like.device:
        raise ValueError(f"workspace: memory on {like.device} is wanted")
    return given, given.data_ptr(), given.numel() * given.element_size()


class _on:
    """The device of a tensor made current for a call, and its current stream."""

    def __init__(self, t: torch.Tensor):
        self.guard = torch.cuda.device(t.device) if t.device.index != torch.cuda.current_device() else None
        self.stream = torch.cuda.current_stream(t.device).cuda_stream

    def __enter__(self) -> int:
        if self.guard is not None:
            self.guard.__enter__()
        return self.stream

    def __exit__(self, *exc) -> None:
        if self.guard is not None:
            self.guard.__exit__(*exc)


def top_k(x: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, lse: torch.Tensor | None = None, *,
          temperature: float = 1.0, workspace: torch.Tensor | None = None) -> None:
    """Run rmi_top_k on the current torch stream: the k = values.shape[1] elements of every row of
    `x` that rank first (int32 `indices`), and log(sum(exp(x / temperature))) of every row."""
    lib = api.load()
    d, n_rows, n_cols, ld = _logits(x)
    k = values.shape[-1]
    vp = _ptr(values, (n_rows, k), x.dtype, x, "values")
    ip = _ptr(indices, (n_rows, k), torch.int32, x, "indices")
    lp = _ptr(lse, (n_rows,), torch.float32, x, "lse")
    with _on(x) as stream:
        _, wp, wn = _workspace(workspace, lib.rmi_top_k_workspace_bytes(d, n_rows, n_cols, k), x)
        rc = lib.rmi_top_k(d, n_rows, n_cols, ld, k, temperature, x.data_ptr(), vp, ip, lp, wp, wn, stream)
    if rc != api.OK:
        raise RmiError(rc, "rmi_top_k")


def _teacher(x: torch.Tensor, t_values, t_indices, teacher_lse, row_grad) -> tuple:
    n_rows, k = x.shape[0], t_values.shape[-1]
    return (_dtype_of(t_values, "t_values"), k, _ptr(t_values, (n_rows, k), t_values.dtype, x, "t_values"),
            _ptr(t_indices, (n_rows, k), torch.int32, x, "t_indices"),
            _ptr(teacher_lse, (n_rows,), torch.float32, x, "teacher_lse"),
            _ptr(row_grad, (n_rows,), torch.float32, x, "row_grad"))


def _grad(x: torch.Tensor, grad: torch.Tensor) -> tuple[int, int]:
    if grad.dtype != x.dtype or grad.shape != x.shape or grad.device != x.device:
        raise ValueError("grad: the type, shape and device of the logits are wanted")
    return grad.data_ptr(), _logits(grad, "grad")[3]


def distill_loss(x: torch.Tensor, t_values: torch.Tensor, t_indices: torch.Tensor, loss: torch.Tensor,
                 stats: torch.Tensor | None = None, grad: torch.Tensor | None = None, *, temperature: float = 1.0,
                 scale: float = 1.0, teacher_lse: torch.Tensor | None = None, row_grad: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None) -> None:
    """Run rmi_distill_loss on the current torch stream: the loss of every row of student logits
    against a teacher's stored best logits; `stats` ([rows, 2]) for distill_grad, or the gradient at
    once in `grad`, which may be `x`."""
    lib = api.load()
    d, n_rows, n_cols, ld = _logits(x)
    td, k, tv, ti, tl, rg = _teacher(x, t_values, t_indices, teacher_lse, row_grad)
    lp = _ptr(loss, (n_rows,), torch.float32, x, "loss")
    sp = _ptr(stats, (n_rows, 2), torch.float32, x, "stats")
    gp, ldg = _grad(x, grad) if grad is not None else (None, 0)
    with _on(x) as stream:
        _, wp, wn = _workspace(workspace, lib.rmi_distill_workspace_bytes(d, n_rows, n_cols, k), x)
        rc = lib.rmi_distill_loss(d, td, n_rows, n_cols, ld, k, temperature, scale, x.data_ptr(), tv, ti, tl, lp, sp,
                                  rg, gp, ldg, wp, wn, stream)
    if rc != api.OK:
        raise RmiError(rc, "rmi_distill_loss")


def distill_grad(x: torch.Tensor, t_values: torch.Tensor, t_indices: torch.Tensor, stats: torch.Tensor,
                 grad: torch.Tensor, *, temperature: float = 1.0, scale: float = 1.0,
                 teacher_lse: torch.Tensor | None = None, row_grad: torch.Tensor | None = None) -> None:
    """Run rmi_distill_grad on the current torch stream: the gradient of an earlier distill_loss from
    its `stats`, for the gradient `row_grad` of every row's loss (None: ones)."""
    lib = api.load()
    d, n_rows, n_cols, ld = _logits(x)
    td, k, tv, ti, tl, rg = _teacher(x, t_values, t_indices, teacher_lse, row_grad)
    sp = _ptr(stats, (n_rows, 2), torch.float32, x, "stats")
    gp, ldg = _grad(x, grad)
    with _on(x) as stream:
        rc = lib.rmi_distill_grad(d, td, n_rows, n_cols, ld, k, temperature, scale, x.data_ptr(), tv, ti, tl, sp, rg,
                                  gp, ldg, stream)
    if rc != api.OK:
        raise RmiError(rc, "rmi_distill_grad")


def sample(x: torch.Tensor, u: torch.Tensor, token: torch.Tensor, logprob: torch.Tensor | None = None, *,
           temperature: torch.Tensor | None = None, top_k: torch.Tensor | None = None,
           top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           allowed: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> None:
    """Run rmi_sample on the current torch stream: one int32 `token` of every row of `x` for the
    random numbers `u`, with one setting per row (`top_k` int32, the others float32), and among the
    tokens whose bit is set in `allowed` ([rows, ceil(vocabulary / 32)] int32 or uint32 words)."""
    lib = api.load()
    d, n_rows, n_cols, ld = _logits(x)
    per_row = (n_rows,)
    ap, lda = None, 0
    if allowed is not None:
        words = (n_cols + 31) // 32
        if (allowed.dtype not in (torch.int32, torch.uint32) or allowed.shape != (n_rows, words)
                or (allowed.stride(1) != 1 and words > 1) or (n_rows > 1 and allowed.stride(0) < words)
                or allowed.device != x.device):
            raise ValueError(f"allowed: [{n_rows}, {words}] 32-bit words on {x.device} are wanted")
        ap, lda = allowed.data_ptr(), max(allowed.stride(0), words)
    args = (_ptr(temperature, per_row, torch.float32, x, "temperature"), _ptr(top_k, per_row, torch.int32, x, "top_k"),
            _ptr(top_p, per_row, torch.float32, x, "top_p"), _ptr(min_p, per_row, torch.float32, x, "min_p"),
            _ptr(u, per_row, torch.float32, x, "u"), _ptr(token, per_row, torch.int32, x, "token"),
            _ptr(logprob, per_row, torch.float32, x, "logprob"))
    with _on(x) as stream:
        _, wp, wn = _workspace(workspace, lib.rmi_sample_workspace_bytes(d, n_rows, n_cols), x)
        rc = lib.rmi_sample(d, n_rows, n_cols, ld, x.data_ptr(), ap, lda, *args, wp, wn, stream)
    if rc != api.OK:
        raise RmiError(rc, "rmi_sample")
