"""Python binding of libdflashcuda.so (ctypes over the C ABI in include/dflash_cuda.h).

Torch is used here only as device-memory and stream plumbing: tensors are handed to the
library as raw device pointers together with the current CUDA stream.  Every compute
call goes to the CUDA library; there is no CPU path.  If the shared library is missing
the import fails loudly.

Reference interface mirrored (random1st/dflash-swift):
  * ``SmallMQuantizedMatmul`` (Sources/DFlashKit/SmallMQuantizedMatmul.swift:27-225):
    ``apply``, ``is_eligible``, ``tiles``, row-count constants.
  * ``SmallMQuantizedLinear`` (:234-293): a quantized linear layer whose call routes
    through the kernel, sharing (never copying) the layer's packed arrays.
  * ``enable_small_m_quantized_matmul`` (:304-317): swaps every eligible layer of a
    module tree and returns how many were swapped (idempotent).
  * The gated-delta capture/replay used by rollbackGatedDeltaRound/Tree
    (DFlashSpeculativeGenerator.swift:450-461): ``gdn_step``, ``gdn_replay``,
    ``gdn_conv_rollback``.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path
from typing import Optional, Sequence

HERE = Path(__file__).resolve().parent
LIB_PATH = Path(os.environ.get("DFLASH_CUDA_LIB", HERE / "libdflashcuda.so"))

DFLASH_OK = 0
DFLASH_ERR_INVALID_ARGUMENT = 1
DFLASH_ERR_UNSUPPORTED = 2
DFLASH_ERR_MISALIGNED = 3
DFLASH_ERR_CUDA = 4
DFLASH_ERR_NCCL = 5
DFLASH_ERR_TIMEOUT = 6
DFLASH_ERR_WORKSPACE = 7

DEVERR_QMM_PIPELINE = 0x1
DEVERR_QMM_REDUCE = 0x2
DEVERR_ALLREDUCE = 0x4
DEVERR_POSITION = 0x8
DEVERR_ATTN_PIPELINE = 0x10
DEVERR_TEST_WAIT = 0x80000000

# Every symbol the header declares; tests check the library exports all of them.
EXPORTED = (
    "dflash_version", "dflash_last_error", "dflash_status_string", "dflash_device_error",
    "dflash_test_bounded_wait", "dflash_qmm_workspace_bytes", "dflash_qmm", "dflash_qmm_noalloc",
    "dflash_qmm_supported", "dflash_qmm_host_workspace_bytes", "dflash_qmm_host", "dflash_bias_add",
    "dflash_gdn_step", "dflash_gdn_replay", "dflash_gdn_conv_rollback",
    # include/dflash_stack.h: glue of the tensor-parallel verify stack
    "dflash_stack_add_rmsnorm", "dflash_stack_silu_mul", "dflash_stack_conv_silu", "dflash_stack_gdn_gates",
    "dflash_stack_gated_norm", "dflash_stack_attn_prep", "dflash_stack_attn_decode",
    "dflash_stack_add_rmsnorm_reduce", "dflash_tp_exchange_bytes", "dflash_tp_exchange_alloc",
    "dflash_tp_exchange_free", "dflash_ipc_get_handle", "dflash_ipc_open_handle", "dflash_ipc_close_handle",
    "dflash_tp_push", "dflash_qmm_ex", "dflash_accept", "dflash_stack_gdn_conv_gates",
    "dflash_accept_reduce",
    # speculative tree rounds
    "dflash_gdn_step_tree", "dflash_stack_gdn_conv_gates_tree", "dflash_stack_attn_prep_tree",
    "dflash_stack_attn_decode_tree", "dflash_stack_kv_compact", "dflash_accept_tree",
    # gated-delta layers with shared key heads
    "dflash_gdn_step_grouped", "dflash_gdn_step_tree_grouped", "dflash_gdn_replay_grouped",
    "dflash_stack_gdn_conv_gates_grouped",
    # attention with a device-resident cache position
    "dflash_stack_attn_prep_ex", "dflash_stack_attn_decode_ex",
    # the verify stack as one object
    "dflash_stack_create", "dflash_stack_forward", "dflash_stack_verify", "dflash_stack_commit",
    "dflash_stack_advance", "dflash_stack_context", "dflash_stack_output", "dflash_stack_destroy",
    # include/dflash_batch.h: batches of sequences, quantised caches, a shared prefix, log probabilities
    "dflash_stack_attn_prep_batch", "dflash_stack_kv_read", "dflash_stack_kv_write", "dflash_stack_kv_compact_batch",
    "dflash_stack_attn_decode_batch", "dflash_stack_attn_decode_batch_workspace_bytes", "dflash_logprobs",
)


class DFlashError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"status {status}: {message}")
        self.status = status


_vp = ctypes.c_void_p
_i = ctypes.c_int
_sz = ctypes.c_size_t
_f = ctypes.c_float
_ll = ctypes.c_longlong


def _load() -> ctypes.CDLL:
    if not LIB_PATH.exists():
        raise ImportError(
            f"libdflashcuda.so not found at {LIB_PATH}; build it with `python -c "
            f"'import __graft_entry__ as g; g.build()'` (no CPU fallback exists)")
    lib = ctypes.CDLL(str(LIB_PATH))
    sig = {
        "dflash_version": ([], _i),
        "dflash_last_error": ([], ctypes.c_char_p),
        "dflash_status_string": ([_i], ctypes.c_char_p),
        "dflash_device_error": ([ctypes.POINTER(ctypes.c_uint32), _vp], _i),
        "dflash_test_bounded_wait": ([ctypes.c_uint64, _vp], _i),
        "dflash_qmm_workspace_bytes": ([_i, _i, _i, _i, _i], _sz),
        "dflash_qmm": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp, _sz, _vp], _i),
        "dflash_qmm_noalloc": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp], _i),
        "dflash_qmm_supported": ([_i, _i, _i, _i], _i),
        "dflash_qmm_host_workspace_bytes": ([_i, _i, _i, _i, _i], _sz),
        "dflash_bias_add": ([_vp, _vp, _i, _i, _vp], _i),
        "dflash_qmm_host": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp, _sz, _vp], _i),
        "dflash_gdn_step": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, ctypes.c_float, _vp], _i),
        "dflash_gdn_replay": ([_vp, _vp, _vp, _vp, _vp, _vp, ctypes.POINTER(ctypes.c_int32), _i, _i, _i, _i,
                               _i, _i, _vp], _i),
        "dflash_gdn_conv_rollback": ([_vp, _vp, _vp, ctypes.POINTER(ctypes.c_int32), _i, _i, _i, _i, _i, _vp],
                                     _i),
        "dflash_stack_add_rmsnorm": ([_vp, _vp, _vp, _vp, _i, _i, _f, _vp], _i),
        "dflash_stack_silu_mul": ([_vp, _vp, _i, _i, _vp], _i),
        "dflash_stack_conv_silu": ([_vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _vp], _i),
        "dflash_stack_gdn_gates": ([_vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _vp], _i),
        "dflash_stack_gated_norm": ([_vp, _vp, _i, _vp, _vp, _i, _i, _i, _f, _vp], _i),
        "dflash_stack_attn_prep": ([_vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _f, _f, _vp], _i),
        "dflash_stack_attn_decode": ([_vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _f, _vp], _i),
        "dflash_stack_add_rmsnorm_reduce": ([_vp, _vp, _i, _i, _vp, _vp, _i, _i, _f, _vp], _i),
        "dflash_tp_exchange_bytes": ([_i, _i, _i], _sz),
        "dflash_tp_exchange_alloc": ([_sz, ctypes.POINTER(_vp)], _i),
        "dflash_tp_exchange_free": ([_vp], _i),
        "dflash_ipc_get_handle": ([_vp, _vp], _i),
        "dflash_ipc_open_handle": ([_vp, ctypes.POINTER(_vp)], _i),
        "dflash_ipc_close_handle": ([_vp], _i),
        "dflash_tp_push": ([_vp, ctypes.POINTER(_vp), _i, _i, _i, _i, _i, _vp], _i),
        "dflash_qmm_ex": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp, _sz, ctypes.c_void_p, _vp], _i),
        "dflash_accept": ([_vp, _vp, _i, _vp, _vp, _vp], _i),
        "dflash_accept_reduce": ([_vp, _i, _i, _vp, _i, _vp, _vp, _vp], _i),
        "dflash_stack_gdn_conv_gates": ([_vp, _i, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp],
                                        _i),
        "dflash_gdn_step_tree": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _vp], _i),
        "dflash_stack_gdn_conv_gates_tree": ([_vp, _i, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i,
                                              _vp, _vp], _i),
        "dflash_stack_attn_prep_tree": ([_vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _f, _f, _vp, _vp],
                                        _i),
        "dflash_stack_attn_decode_tree": ([_vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _f, _vp, _vp], _i),
        "dflash_stack_kv_compact": ([_vp, _vp, _i, ctypes.c_longlong, _i, _i, _i, _i,
                                     ctypes.POINTER(ctypes.c_int32), _i, _vp], _i),
        "dflash_accept_tree": ([_vp, _vp, _vp, _i, _vp, _vp, _vp, _vp], _i),
        "dflash_gdn_step_grouped": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _f, _vp], _i),
        "dflash_gdn_step_tree_grouped": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _f, _vp], _i),
        "dflash_gdn_replay_grouped": ([_vp, _vp, _vp, _vp, _vp, _vp, ctypes.POINTER(ctypes.c_int32), _i, _i, _i, _i,
                                       _i, _i, _i, _vp], _i),
        "dflash_stack_gdn_conv_gates_grouped": ([_vp, _i, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i,
                                                 _i, _vp, _vp], _i),
        "dflash_stack_attn_prep_ex": ([_vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _f, _f, _vp, _vp, _vp],
                                      _i),
        "dflash_stack_attn_decode_ex": ([_vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _f, _vp, _vp, _vp], _i),
        "dflash_stack_create": ([_vp, _i, ctypes.POINTER(_vp)], _i),
        "dflash_stack_forward": ([_vp, _vp, _vp, _vp], _i),
        "dflash_stack_verify": ([_vp, _vp, _vp, _vp, _vp, _vp], _i),
        "dflash_stack_commit": ([_vp, ctypes.POINTER(ctypes.c_int32), _i, _vp], _i),
        "dflash_stack_advance": ([_vp, _i], _i),
        "dflash_stack_context": ([_vp], _i),
        "dflash_stack_output": ([_vp], _vp),
        "dflash_stack_destroy": ([_vp], None),
        "dflash_stack_attn_prep_batch": ([_vp, _ll, _vp, _vp, _vp, _ll, _vp, _vp, _i, _i, _i, _i, _f, _f, _vp, _vp], _i),
        "dflash_stack_kv_read": ([_vp, _vp, _i, _vp, _vp, _vp], _i),
        "dflash_stack_kv_write": ([_vp, _vp, _i, _vp, _vp, _vp], _i),
        "dflash_stack_kv_compact_batch": ([_vp, _vp, _vp, _vp, _i, _vp], _i),
        "dflash_stack_attn_decode_batch_workspace_bytes": ([_vp, _i, _i, _i], _sz),
        "dflash_stack_attn_decode_batch": ([_vp, _ll, _vp, _ll, _vp, _vp, _vp, _i, _vp, _i, _i, _f, _vp, _vp, _sz, _vp],
                                           _i),
        "dflash_logprobs": ([_vp, _i, _ll, _i, _i, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp], _i),
    }
    for name, (args, res) in sig.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    return lib


lib = _load()


def last_error() -> str:
    return lib.dflash_last_error().decode()


def check(status: int) -> None:
    if status != DFLASH_OK:
        raise DFlashError(status, last_error())


def _stream(stream=None) -> int:
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
    return stream.cuda_stream


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def device_error(stream=None) -> int:
    """Reads and clears the device error word (synchronises the stream)."""
    bits = ctypes.c_uint32(0)
    check(lib.dflash_device_error(ctypes.byref(bits), _stream(stream)))
    return int(bits.value)


def test_bounded_wait(limit_ns: int, stream=None) -> None:
    check(lib.dflash_test_bounded_wait(int(limit_ns), _stream(stream)))


# ----------------------------------------------------------------------------- qmm

def qmm_workspace_bytes(M: int, N: int, K: int, group_size: int, bits: int) -> int:
    return int(lib.dflash_qmm_workspace_bytes(M, N, K, group_size, bits))


class Workspace:
    """Zero-initialised device workspace for dflash_qmm (one per stream)."""

    def __init__(self, nbytes: int, device=None):
        import torch
        self.nbytes = int(nbytes)
        self.buf = torch.zeros(max(self.nbytes, 16), dtype=torch.uint8, device=device or "cuda")

    def ensure(self, nbytes: int) -> "Workspace":
        if nbytes > self.nbytes:
            self.__init__(nbytes, self.buf.device)
        return self


_workspaces: dict = {}


def default_workspace(nbytes: int, device) -> Workspace:
    import torch
    key = (str(device), torch.cuda.current_stream(device).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = Workspace(nbytes, device)
    return ws.ensure(nbytes)


def qmm(x, w, scales, biases, group_size: int, bits: int, out=None, workspace: Optional[Workspace] = None,
        stream=None):
    """y = x . dequant(w)^T through dflash_qmm.  x: bf16 [M, K] (M <= 16) on the GPU."""
    import torch
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    need = qmm_workspace_bytes(M, N, K, group_size, bits)
    ws = workspace.ensure(need) if workspace is not None else default_workspace(need, x.device)
    check(lib.dflash_qmm(_ptr(x), _ptr(w), _ptr(scales), _ptr(biases), _ptr(out), M, N, K, group_size, bits,
                         ws.buf.data_ptr(), ws.nbytes, _stream(stream)))
    return out


def qmm_host_workspace_bytes(M: int, N: int, K: int, group_size: int, bits: int) -> int:
    return int(lib.dflash_qmm_host_workspace_bytes(M, N, K, group_size, bits))


def qmm_host(x_host, w, scales, biases, group_size: int, bits: int, out_host=None,
             workspace: Optional[Workspace] = None, stream=None):
    """dflash_qmm_host: x bf16 [M, K] and the result in HOST memory (pinned for
    asynchronous copies), weights on the GPU; one library call queues copy in, matmul
    and copy out on the stream.  The result is valid after the stream has run past it."""
    import torch
    M, K = x_host.shape
    N = w.shape[0]
    if out_host is None:
        out_host = torch.empty((M, N), dtype=torch.bfloat16).pin_memory()
    need = qmm_host_workspace_bytes(M, N, K, group_size, bits)
    ws = workspace.ensure(need) if workspace is not None else default_workspace(need, w.device)
    check(lib.dflash_qmm_host(_ptr(x_host), _ptr(w), _ptr(scales), _ptr(biases), _ptr(out_host), M, N, K, group_size,
                              bits, ws.buf.data_ptr(), ws.nbytes, _stream(stream)))
    return out_host


def qmm_noalloc(x, w, scales, biases, group_size: int, bits: int, out=None, stream=None):
    """dflash_qmm without a workspace argument, for callers that may not allocate
    device memory: the library's own static device scratch is used instead (shapes up
    to its 8 MiB limit).  Calls on one device share the scratch: keep them ordered on
    one stream, or use qmm with one workspace per stream."""
    import torch
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    check(lib.dflash_qmm_noalloc(_ptr(x), _ptr(w), _ptr(scales), _ptr(biases), _ptr(out), M, N, K, group_size, bits,
                                 _stream(stream)))
    return out


class SmallMQuantizedMatmul:
    """Constants and dispatch of the small-M kernel (SmallMQuantizedMatmul.swift:27-225).

    The reference kernel only wins from 6 rows (below that MLX's GEMV is at roofline,
    :29-32) and stops at 16 (two 8-row MMA tiles, :36-37).  This library has no stock
    op to defer to, so its kernel covers every row count 1..16; wider inputs are cut
    into 16-row passes by SmallMQuantizedLinear.
    """

    minimum_rows = 1
    maximum_rows = 16
    rows_per_tile = 8
    supported_bits = (4, 8)
    supported_group_sizes = (32, 64, 128)

    @staticmethod
    def is_eligible(layer: "QuantizedLinear") -> bool:
        """Static half of the test (SmallMQuantizedMatmul.swift:193-201): affine mode
        with biases, a bit width and group size the kernel covers, and a shape it can
        tile."""
        if getattr(layer, "mode", "affine") != "affine" or layer.biases is None:
            return False
        out_features, in_features = layer.shape
        return bool(lib.dflash_qmm_supported(out_features, in_features, layer.group_size, layer.bits))

    @staticmethod
    def tiles(rows: int) -> int:
        """MMA n-tiles needed for `rows` (SmallMQuantizedMatmul.swift:205-207)."""
        return 1 if rows <= SmallMQuantizedMatmul.rows_per_tile else 2

    @staticmethod
    def apply(x, weight, scales, biases, rows: int, output_features: int, input_features: int, bits: int,
              group_size: int = 64):
        """x[rows, K] . deq(weight)^T -> [rows, N] bf16 (SmallMQuantizedMatmul.swift:210-224)."""
        assert x.shape[0] == rows and x.shape[1] == input_features and weight.shape[0] == output_features
        return qmm(x, weight, scales, biases, group_size, bits)


class QuantizedLinear:
    """MLX-layout affine-quantized linear layer: packed uint32 weight [N, K*bits/32],
    bf16 scales and biases [N, K/group_size], optional bf16 bias [N]."""

    def __init__(self, weight, scales, biases, group_size: int, bits: int, bias=None, mode: str = "affine"):
        self.weight, self.scales, self.biases, self.bias = weight, scales, biases, bias
        self.group_size, self.bits, self.mode = int(group_size), int(bits), mode
        self.frozen = False

    @property
    def shape(self):
        return (self.weight.shape[0], self.weight.shape[1] * 32 // self.bits)

    def freeze(self):
        self.frozen = True
        return self

    def __call__(self, x):
        raise NotImplementedError("the stock MLX quantizedMatmul is not part of this library; "
                                  "wrap the layer in SmallMQuantizedLinear")


class SmallMQuantizedLinear(QuantizedLinear):
    """QuantizedLinear whose forward runs on dflash_qmm (SmallMQuantizedMatmul.swift:234-293).

    Shares the wrapped layer's arrays (no copy) and stays frozen like the layer it
    replaces (:243-252).  The call flattens leading dimensions to rows (:255-256,
    :270), runs the kernel in passes of at most 16 rows (the kernel reads x rows in
    place, so the reference's zero-padding concat of :271-281 is not needed), reshapes
    back and adds the optional bias (:287-290).  Only bf16 input is accepted: the
    kernel's fragments and output are bf16 (:257-263); other dtypes raise TypeError
    rather than silently change the layer's output dtype.
    """

    def __init__(self, other: QuantizedLinear):
        super().__init__(other.weight, other.scales, other.biases, other.group_size, other.bits,
                         bias=other.bias, mode=other.mode)
        self.kernel_eligible = SmallMQuantizedMatmul.is_eligible(other)
        self.freeze()

    def __call__(self, x, stream=None):
        import torch
        if not self.kernel_eligible:
            raise DFlashError(DFLASH_ERR_UNSUPPORTED,
                              f"layer {self.shape} bits={self.bits} group={self.group_size} is not covered")
        if x.dtype != torch.bfloat16:
            raise TypeError(f"SmallMQuantizedLinear takes bfloat16 input, got {x.dtype}")
        lead = x.shape[:-1]
        K = x.shape[-1]
        N = self.weight.shape[0]
        flat = x.reshape(-1, K)
        if not flat.is_contiguous():
            flat = flat.contiguous()
        rows = flat.shape[0]
        y = torch.empty((rows, N), dtype=torch.bfloat16, device=x.device)
        step = SmallMQuantizedMatmul.maximum_rows
        for r0 in range(0, rows, step):
            r1 = min(rows, r0 + step)
            qmm(flat[r0:r1], self.weight, self.scales, self.biases, self.group_size, self.bits, out=y[r0:r1],
                stream=stream)
        if self.bias is not None and rows > 0:
            check(lib.dflash_bias_add(_ptr(y), _ptr(self.bias), rows, N, _stream(stream)))
        return y.reshape(*lead, N)


def enable_small_m_quantized_matmul(model) -> int:
    """Swaps every eligible QuantizedLinear in `model` for a SmallMQuantizedLinear
    (SmallMQuantizedMatmul.swift:304-317).  `model` is any object tree whose
    attributes (or list/dict items) hold layers.  Returns the number swapped; a second
    call returns 0 because wrapped layers are never wrapped again."""
    count = 0

    def visit(obj, seen):
        nonlocal count
        if id(obj) in seen:
            return
        seen.add(id(obj))
        items = []
        if isinstance(obj, dict):
            items = list(obj.items())
        elif isinstance(obj, (list, tuple)):
            items = list(enumerate(obj))
        elif hasattr(obj, "__dict__"):
            items = list(vars(obj).items())
        for key, child in items:
            if isinstance(child, QuantizedLinear):
                if isinstance(child, SmallMQuantizedLinear) or not SmallMQuantizedMatmul.is_eligible(child):
                    continue
                wrapped = SmallMQuantizedLinear(child)
                if isinstance(obj, dict):
                    obj[key] = wrapped
                elif isinstance(obj, list):
                    obj[key] = wrapped
                elif isinstance(obj, tuple):
                    continue
                else:
                    setattr(obj, key, wrapped)
                count += 1
            elif isinstance(child, (dict, list, tuple)) or (hasattr(child, "__dict__") and not _is_tensor(child)):
                visit(child, seen)

    visit(model, set())
    return count


def _is_tensor(obj) -> bool:
    return type(obj).__module__.startswith("torch")


# ----------------------------------------------------------------------------- gated delta

def gdn_step(state_in, state_out, q, k, v, alpha, beta, out=None, q_scale: float = 1.0, stream=None):
    """One layer's recurrence over T positions (the verify forward; its inputs are the capture).
    q, k [T, Hk, dk]; v [T, H, dv]: Hk < H shares each key head between H / Hk value heads."""
    T, Hk, dk = k.shape
    H, dv = v.shape[-2], v.shape[-1]
    args = (_ptr(state_in), _ptr(state_out), _ptr(q), _ptr(k), _ptr(v), _ptr(alpha), _ptr(beta), _ptr(out), T, H)
    if Hk == H:
        check(lib.dflash_gdn_step(*args, dk, dv, float(q_scale), _stream(stream)))
    else:
        check(lib.dflash_gdn_step_grouped(*args, Hk, dk, dv, float(q_scale), _stream(stream)))
    return state_out


def gdn_step_tree(state_in, q, k, v, alpha, beta, parents, out, q_scale: float = 1.0, stream=None):
    """One layer's recurrence over the T rows of a tree round: row t gets the output of a
    chain over its root-to-t path from state_in.  parents: device int32 [T].  Key heads as
    for gdn_step."""
    T, Hk, dk = k.shape
    H, dv = v.shape[-2], v.shape[-1]
    args = (_ptr(state_in), _ptr(q), _ptr(k), _ptr(v), _ptr(alpha), _ptr(beta), _ptr(parents), _ptr(out), T, H)
    if Hk == H:
        check(lib.dflash_gdn_step_tree(*args, dk, dv, float(q_scale), _stream(stream)))
    else:
        check(lib.dflash_gdn_step_tree_grouped(*args, Hk, dk, dv, float(q_scale), _stream(stream)))
    return out


def _rows_arg(rows: Optional[Sequence[int]]):
    if rows is None:
        return None
    arr = (ctypes.c_int32 * len(rows))(*[int(r) for r in rows])
    return arr


def gdn_replay(snapshot, state_out, k, v, alpha, beta, keep: int, rows: Optional[Sequence[int]] = None,
               stream=None):
    """Rollback replay for all layers at once.  k: [L, width, Hk, dk]; v: [L, width, H, dv];
    state: [L, H, dv, dk] (Hk < H: shared key heads, as for gdn_step)."""
    L, width, Hk, dk = k.shape
    H, dv = v.shape[-2], v.shape[-1]
    if rows is not None and len(rows) < keep:
        raise ValueError("rows shorter than keep")
    args = (_ptr(snapshot), _ptr(state_out), _ptr(k), _ptr(v), _ptr(alpha), _ptr(beta), _rows_arg(rows), int(keep),
            width, L, H)
    if Hk == H:
        check(lib.dflash_gdn_replay(*args, dk, dv, _stream(stream)))
    else:
        check(lib.dflash_gdn_replay_grouped(*args, Hk, dk, dv, _stream(stream)))
    return state_out


def gdn_conv_rollback(window, window_out, conv_in, keep: int, rows: Optional[Sequence[int]] = None, stream=None):
    """Conv-window rebuild.  window: [L, kc1, C]; conv_in: [L, width, C]."""
    L, kc1, C = window.shape
    width = conv_in.shape[1]
    if rows is not None and len(rows) < keep:
        raise ValueError("rows shorter than keep")
    check(lib.dflash_gdn_conv_rollback(_ptr(window), _ptr(window_out), _ptr(conv_in), _rows_arg(rows), int(keep),
                                       width, L, kc1, C, _stream(stream)))
    return window_out


# ----------------------------------------------------------------------------- verify-stack glue
# (include/dflash_stack.h; tensors row-major with one row per token)

def stack_add_rmsnorm(resid, delta, weight, out, eps: float, stream=None):
    M, H = resid.shape
    check(lib.dflash_stack_add_rmsnorm(_ptr(resid), _ptr(delta), _ptr(weight), _ptr(out), M, H, float(eps),
                                       _stream(stream)))
    return out


def stack_silu_mul(gate_up, out, stream=None):
    M, I = out.shape
    check(lib.dflash_stack_silu_mul(_ptr(gate_up), _ptr(out), M, I, _stream(stream)))
    return out


def stack_conv_silu(x, window, weight, out, channels: int, parts: int, stream=None):
    """x: [M, ld] (channels convolved at [0, channels)); window [kc-1, C]; out [parts, M, C/parts]."""
    M, ld = x.shape[0], x.stride(0)
    kc = weight.shape[1]
    check(lib.dflash_stack_conv_silu(_ptr(x), ld, _ptr(window), _ptr(weight), _ptr(out), M, channels, kc, parts,
                                     _stream(stream)))
    return out


def stack_gdn_gates(q, k, ab, a_log, dt_bias, alpha, beta, stream=None):
    """q, k: [M, H, dk] (normalised in place); ab: [M, ld] with b then a; alpha, beta [M, H] fp32."""
    M, H, dk = q.shape
    check(lib.dflash_stack_gdn_gates(_ptr(q), _ptr(k), _ptr(ab), ab.stride(0), _ptr(a_log), _ptr(dt_bias),
                                     _ptr(alpha), _ptr(beta), M, H, dk, _stream(stream)))


def stack_gated_norm(o, z, weight, out, eps: float, stream=None):
    """o: [M, H, dv]; z: [M, >= H*dv] rows; out: [M, H*dv]."""
    M, H, dv = o.shape
    check(lib.dflash_stack_gated_norm(_ptr(o), _ptr(z), z.stride(0), _ptr(weight), _ptr(out), M, H, dv, float(eps),
                                      _stream(stream)))
    return out


def stack_attn_prep(qkv, q_norm, k_norm, cache_k, cache_v, hq: int, hkv: int, rot: int, pos0: int, eps: float,
                    theta: float, stream=None, parents=None, position=None):
    """qkv rows [q | gate | k | v]; caches [hkv, max_len, d].  parents (device int32 [M]):
    a tree round, rotary position pos0 + depth.  position (device int32 [1]): pos0 read on
    the device instead (dflash_stack_attn_prep_ex)."""
    M = qkv.shape[0]
    _, max_len, d = cache_k.shape
    args = (_ptr(qkv), qkv.stride(0), _ptr(q_norm), _ptr(k_norm), _ptr(cache_k), _ptr(cache_v), M, hq, hkv, d, rot,
            pos0, max_len, float(eps), float(theta))
    if position is not None:
        check(lib.dflash_stack_attn_prep_ex(*args, _ptr(parents), _ptr(position), _stream(stream)))
    elif parents is None:
        check(lib.dflash_stack_attn_prep(*args, _stream(stream)))
    else:
        check(lib.dflash_stack_attn_prep_tree(*args, _ptr(parents), _stream(stream)))


def stack_attn_decode(qkv, cache_k, cache_v, out, hq: int, hkv: int, pos0: int, scale: float, stream=None,
                      parents=None, position=None):
    """parents (device int32 [M]): a tree round, each token sees the prefix and its path.
    position (device int32 [1]): pos0 read on the device (dflash_stack_attn_decode_ex)."""
    M = qkv.shape[0]
    _, max_len, d = cache_k.shape
    args = (_ptr(qkv), qkv.stride(0), _ptr(cache_k), _ptr(cache_v), _ptr(out), M, hq, hkv, d, pos0, max_len,
            float(scale))
    if position is not None:
        check(lib.dflash_stack_attn_decode_ex(*args, _ptr(parents), _ptr(position), _stream(stream)))
    elif parents is None:
        check(lib.dflash_stack_attn_decode(*args, _stream(stream)))
    else:
        check(lib.dflash_stack_attn_decode_tree(*args, _ptr(parents), _stream(stream)))
    return out


def accept_tree(target_tokens, parents, tokens, path, path_len, next_token, stream=None):
    """The accepted path of a tree round on the device: target_tokens, parents, tokens
    int32 [rows]; writes path int32 [rows] (first path_len entries), path_len [1],
    next_token [1]."""
    check(lib.dflash_accept_tree(_ptr(target_tokens), _ptr(parents), _ptr(tokens), tokens.shape[0], _ptr(path),
                                 _ptr(path_len), _ptr(next_token), _stream(stream)))


def stack_kv_compact(cache_k, cache_v, pos0: int, rows: Sequence[int], stream=None):
    """After a tree round: cache rows pos0 + rows[i] -> pos0 + i.  Caches [hkv, max_len, d]
    (one layer) or [layers, hkv, max_len, d] (contiguous)."""
    if cache_k.dim() == 3:
        layers, (hkv, max_len, d), stride = 1, cache_k.shape, 0
    else:
        layers, hkv, max_len, d = cache_k.shape
        stride = cache_k.stride(0)
    check(lib.dflash_stack_kv_compact(_ptr(cache_k), _ptr(cache_v), layers, stride, hkv, d, pos0, max_len,
                                      _rows_arg(rows), len(rows), _stream(stream)))


# ----------------------------------------------------------------------------- tensor-parallel exchange

IPC_HANDLE_BYTES = 64


class PeerExchange:
    """This rank's exchange buffer for the peer all-reduce (include/dflash_stack.h), mapped
    into every rank of the node.  `handles` come from ``handle()`` on every rank (the
    host exchanges them, e.g. with torch.distributed.all_gather_object)."""

    def __init__(self, world: int, M: int, H: int):
        self.world, self.M, self.H = world, M, H
        self.nbytes = int(lib.dflash_tp_exchange_bytes(world, M, H))
        if self.nbytes == 0:
            raise DFlashError(DFLASH_ERR_INVALID_ARGUMENT, f"exchange of world {world}, [{M}, {H}] not supported")
        ptr = ctypes.c_void_p()
        check(lib.dflash_tp_exchange_alloc(self.nbytes, ctypes.byref(ptr)))
        self.ptr = ptr.value
        self.bases = None
        self._opened = []

    def handle(self) -> bytes:
        buf = ctypes.create_string_buffer(IPC_HANDLE_BYTES)
        check(lib.dflash_ipc_get_handle(self.ptr, buf))
        return buf.raw

    def connect(self, rank: int, handles) -> None:
        bases = []
        for r, h in enumerate(handles):
            if r == rank:
                bases.append(self.ptr)
                continue
            p = ctypes.c_void_p()
            check(lib.dflash_ipc_open_handle(ctypes.create_string_buffer(bytes(h), IPC_HANDLE_BYTES), ctypes.byref(p)))
            self._opened.append(p.value)
            bases.append(p.value)
        self.rank = rank
        self.bases = (ctypes.c_void_p * len(bases))(*bases)

    def connect_local(self, rank: int, ptrs) -> None:
        """Use buffers of this process as the ranks' buffers (single-process tests)."""
        self.rank = rank
        self.bases = (ctypes.c_void_p * len(ptrs))(*ptrs)

    def push(self, part, set_: int, stream=None) -> None:
        M, H = part.shape
        check(lib.dflash_tp_push(_ptr(part), self.bases, self.rank, self.world, M, H, set_, _stream(stream)))

    def close(self) -> None:
        for p in self._opened:
            lib.dflash_ipc_close_handle(p)
        self._opened = []
        if self.ptr:
            lib.dflash_tp_exchange_free(self.ptr)
            self.ptr = None


def stack_add_rmsnorm_reduce(resid, exchange: PeerExchange, set_: int, weight, out, eps: float, stream=None):
    M, H = resid.shape
    check(lib.dflash_stack_add_rmsnorm_reduce(_ptr(resid), exchange.ptr, exchange.world, set_, _ptr(weight), _ptr(out),
                                              M, H, float(eps), _stream(stream)))
    return out


class QmmOptions(ctypes.Structure):
    """dflash_qmm_options (include/dflash_stack.h)."""
    _fields_ = [("x_swiglu", ctypes.c_int), ("push", ctypes.c_int), ("rank", ctypes.c_int), ("world", ctypes.c_int),
                ("set", ctypes.c_int), ("bases", ctypes.c_void_p), ("argmax_keys", ctypes.c_void_p),
                ("argmax_index_base", ctypes.c_int)]


def qmm_ex(x, w, scales, biases, group_size: int, bits: int, out=None, workspace: Optional[Workspace] = None,
           swiglu: bool = False, exchange: Optional[PeerExchange] = None, set_: int = 0, argmax_keys=None,
           argmax_index_base: int = 0, stream=None):
    """dflash_qmm_ex: with swiglu, x is [M, 2K] = [gate | up]; with an exchange, the result
    is pushed to every rank's exchange slot (set `set_`) instead of written to `out`; with
    argmax_keys (int64 [M] on the device) each row is reduced to its argmax key instead."""
    import torch
    M = x.shape[0]
    K = x.shape[1] // 2 if swiglu else x.shape[1]
    N = w.shape[0]
    if out is None and exchange is None and argmax_keys is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    o = QmmOptions(int(bool(swiglu)), 0, 0, 1, 0, None, _ptr(argmax_keys), int(argmax_index_base))
    if exchange is not None:
        o.push, o.rank, o.world, o.set = 1, exchange.rank, exchange.world, int(set_)
        o.bases = ctypes.cast(exchange.bases, ctypes.c_void_p)
    need = qmm_workspace_bytes(M, N, K, group_size, bits)
    ws = workspace.ensure(need) if workspace is not None else default_workspace(need, x.device)
    check(lib.dflash_qmm_ex(_ptr(x), _ptr(w), _ptr(scales), _ptr(biases), _ptr(out), M, N, K, group_size, bits,
                            ws.buf.data_ptr(), ws.nbytes, ctypes.addressof(o), _stream(stream)))
    return out


def lm_head_argmax(x, w, scales, biases, group_size: int, bits: int, keys=None, workspace=None, index_base: int = 0,
                   stream=None):
    """Argmax keys of x . deq(W)^T per row without writing the logits (int64 [M]); with
    index_base, W is a vocabulary shard starting at that row."""
    import torch
    if keys is None:
        keys = torch.empty(x.shape[0], dtype=torch.int64, device=x.device)
    qmm_ex(x, w, scales, biases, group_size, bits, workspace=workspace, argmax_keys=keys,
           argmax_index_base=index_base, stream=stream)
    return keys


def accept(keys, proposals, tokens=None, accepted=None, stream=None):
    """dflash_accept: (target tokens int32 [drafts + 1], accepted int32 [1]) on the device."""
    import torch
    drafts = proposals.shape[0]
    if tokens is None:
        tokens = torch.empty(drafts + 1, dtype=torch.int32, device=keys.device)
    if accepted is None:
        accepted = torch.empty(1, dtype=torch.int32, device=keys.device)
    check(lib.dflash_accept(_ptr(keys), _ptr(proposals), drafts, _ptr(tokens), _ptr(accepted), _stream(stream)))
    return tokens, accepted


def stack_gdn_conv_gates(x, window, weight, out, ab, a_log, dt_bias, alpha, beta, heads: int, dk: int, stream=None,
                         parents=None, k_heads: Optional[int] = None):
    """Conv + SiLU + q/k normalisation + gates in one kernel; out [3, M, heads, dk].
    parents (device int32 [M]): a tree round, each row convolved along its path.  k_heads
    < heads: q and k have k_heads heads (dflash_stack_gdn_conv_gates_grouped); out then
    holds [q: M x k_heads dk | k: M x k_heads dk | v: M x heads dk] contiguously."""
    M = x.shape[0]
    if k_heads is not None and k_heads != heads:
        check(lib.dflash_stack_gdn_conv_gates_grouped(
            _ptr(x), x.stride(0), _ptr(window), _ptr(weight), _ptr(out), _ptr(ab), ab.stride(0), _ptr(a_log),
            _ptr(dt_bias), _ptr(alpha), _ptr(beta), M, heads, k_heads, dk, weight.shape[1], _ptr(parents),
            _stream(stream)))
        return out
    args = (_ptr(x), x.stride(0), _ptr(window), _ptr(weight), _ptr(out), _ptr(ab), ab.stride(0), _ptr(a_log),
            _ptr(dt_bias), _ptr(alpha), _ptr(beta), M, heads, dk, weight.shape[1])
    if parents is None:
        check(lib.dflash_stack_gdn_conv_gates(*args, _stream(stream)))
    else:
        check(lib.dflash_stack_gdn_conv_gates_tree(*args, _ptr(parents), _stream(stream)))
    return out


def accept_reduce(exchange: PeerExchange, set_: int, proposals, tokens=None, accepted=None, stream=None):
    """dflash_accept_reduce over the ranks' keys pushed into `exchange` (laid out for [M, 4])."""
    import torch
    drafts = proposals.shape[0]
    dev = proposals.device
    if tokens is None:
        tokens = torch.empty(drafts + 1, dtype=torch.int32, device=dev)
    if accepted is None:
        accepted = torch.empty(1, dtype=torch.int32, device=dev)
    check(lib.dflash_accept_reduce(exchange.ptr, exchange.world, int(set_), _ptr(proposals), drafts, _ptr(tokens),
                                   _ptr(accepted), _stream(stream)))
    return tokens, accepted


# ----------------------------------------------------------------------------- batches of sequences
# (include/dflash_batch.h).  A call on tensors of a device that is not the current one, or with
# `stream`, is made with that device and stream current: its outputs and workspace then come
# from that stream's memory.

class KVCacheDesc(ctypes.Structure):
    """dflash_kv_cache."""
    _fields_ = [("k", _vp), ("k_scales", _vp), ("k_biases", _vp), ("v", _vp), ("v_scales", _vp), ("v_biases", _vp),
                ("sequences", _i), ("kv_heads", _i), ("max_len", _i), ("head_dim", _i), ("bits", _i), ("group", _i)]


class KVCache:
    """The attention caches of `sequences` sequences: bits 16 (bf16 rows), or 8 / 4 (affine
    codes with a bf16 scale and bias per `group` elements, the packed layout of the weights).
    k and v are (data, scales, biases), data bf16 [sequences, kv_heads, max_len, head_dim] or
    int32 [sequences, kv_heads, max_len, head_dim * bits / 32]."""

    def __init__(self, sequences: int, kv_heads: int, max_len: int, head_dim: int, bits: int = 16, group: int = 64,
                 device=None):
        import torch
        dev = device or "cuda"

        def one():
            lead = (sequences, kv_heads, max_len)
            if bits == 16:
                return torch.zeros(*lead, head_dim, dtype=torch.bfloat16, device=dev), None, None
            if bits not in (4, 8) or group not in (32, 64, 128) or head_dim % group:
                raise DFlashError(DFLASH_ERR_UNSUPPORTED, f"a {bits}-bit cache in groups of {group} of {head_dim}")
            return (torch.zeros(*lead, head_dim * bits // 32, dtype=torch.int32, device=dev),
                    torch.zeros(*lead, head_dim // group, dtype=torch.bfloat16, device=dev),
                    torch.zeros(*lead, head_dim // group, dtype=torch.bfloat16, device=dev))

        self._bind(one(), one(), bits, group)

    @classmethod
    def of(cls, k, v, bits: int, group: int = 64) -> "KVCache":
        """A cache over tensors that exist: k and v (data, scales, biases), referenced."""
        self = cls.__new__(cls)
        self._bind(k, v, bits, group)
        return self

    def _bind(self, k, v, bits, group):
        import torch
        data = k[0]
        if data.dim() != 4:
            raise ValueError(f"cache data of shape {tuple(data.shape)}: [sequences, kv_heads, max_len, ...] is expected")
        lead = tuple(data.shape[:3])
        head_dim = data.shape[3] if bits == 16 else data.shape[3] * 32 // bits
        for d, s, b in (k, v):
            if d.dtype != (torch.bfloat16 if bits == 16 else torch.int32) or tuple(d.shape) != tuple(data.shape):
                raise ValueError(f"cache data {d.dtype} {tuple(d.shape)} does not fit a {bits}-bit cache like {tuple(data.shape)}")
            parts = (d,) if bits == 16 else (d, s, b)
            for t in parts[1:]:
                if t is None or t.dtype != torch.bfloat16 or tuple(t.shape) != lead + (head_dim // group,):
                    raise ValueError(f"a {bits}-bit cache needs bf16 scales and biases {lead + (head_dim // group,)}")
            if any(not t.is_contiguous() or t.device != data.device for t in parts):
                raise ValueError("the tensors of a cache must be contiguous and on one device")
        self.k, self.v, self.bits, self.group = tuple(k), tuple(v), int(bits), int(group) if bits != 16 else 0
        (self.sequences, self.kv_heads, self.max_len), self.head_dim = lead, int(head_dim)
        self.device = data.device
        p = [_ptr(t) for t in (self.k if bits != 16 else (k[0], None, None)) + (self.v if bits != 16 else (v[0], None, None))]
        self.desc = KVCacheDesc(*p, *lead, self.head_dim, self.bits, self.group)
        self.ref = ctypes.addressof(self.desc)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.k + self.v if t is not None)


def _elsewhere(device, stream):
    """The context in which a call on tensors of `device` has to run, or None for the current one."""
    import torch
    if device.type != "cuda":
        raise ValueError(f"tensors on {device}: the library runs on CUDA devices only")
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"a stream of {stream.device} for tensors on {device}")
        return torch.cuda.stream(stream)
    if device.index != torch.cuda.current_device():
        return torch.cuda.device(device)
    return None


def _current_stream() -> int:
    """The current device's current stream, without the Stream object that torch.cuda.current_stream() makes."""
    import torch
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _rows_bf16(name, t, device, cols=None):
    """Checks rows of bf16 whose elements are adjacent."""
    import torch
    if t.dtype != torch.bfloat16 or t.dim() != 2 or t.stride(1) != 1 or t.device != device or (
            cols is not None and t.shape[1] != cols):
        raise ValueError(f"{name}: bf16 rows on {device} with adjacent elements are expected, got {t.dtype} "
                         f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _ints(name, t, device, shape):
    import torch
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: contiguous int32 {shape} on {device} is expected, got {t.dtype} {tuple(t.shape)} on "
                         f"{t.device}")


def _block_tokens(name, rows: int, cache: KVCache) -> int:
    if rows == 0 or rows % cache.sequences:
        raise ValueError(f"{name}: {rows} rows for {cache.sequences} sequences")
    return rows // cache.sequences


def stack_attn_prep_batch(qkv, q_norm, k_norm, cache: KVCache, lengths, hq: int, rot: int, eps: float, theta: float,
                          q_out=None, position0: int = 0, parents=None, stream=None):
    """Norm and rotary embedding of every sequence's block rows; k and v go to the cache in its
    format at rows lengths[b] + t, the q heads to q_out bf16 [rows, hq * d] (returned).  qkv
    rows [q | gate | k | v], row b * T + t being token t of sequence b; lengths int32
    [sequences] on the device (negative: the sequence takes no part); parents int32
    [sequences, T]: each block is a tree."""
    import torch
    ctx = _elsewhere(cache.device, stream)
    if ctx is not None:
        with ctx:
            return stack_attn_prep_batch(qkv, q_norm, k_norm, cache, lengths, hq, rot, eps, theta, q_out, position0,
                                         parents)
    dev, d = cache.device, cache.head_dim
    T = _block_tokens("qkv", qkv.shape[0], cache)
    _rows_bf16("qkv", qkv, dev)
    if qkv.shape[1] < (2 * hq + 2 * cache.kv_heads) * d:
        raise ValueError(f"qkv rows of {qkv.shape[1]} elements for {hq} q heads and {cache.kv_heads} kv heads of {d}")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w.dtype != torch.bfloat16 or tuple(w.shape) != (d,) or w.stride(0) != 1 or w.device != dev:
            raise ValueError(f"{name}: bf16 [{d}] on {dev} is expected")
    _ints("lengths", lengths, dev, (cache.sequences,))
    if parents is not None:
        _ints("parents", parents, dev, (cache.sequences, T))
    if q_out is None:
        q_out = qkv.new_empty((qkv.shape[0], hq * d))
    else:
        _rows_bf16("q_out", q_out, dev)
        if q_out.shape[0] != qkv.shape[0] or q_out.shape[1] < hq * d:
            raise ValueError(f"q_out {tuple(q_out.shape)} for {qkv.shape[0]} rows of {hq * d}")
    check(lib.dflash_stack_attn_prep_batch(_ptr(qkv), qkv.stride(0), _ptr(q_norm), _ptr(k_norm), _ptr(q_out),
                                           q_out.stride(0), cache.ref, _ptr(lengths), T, hq, rot, position0, eps, theta,
                                           _ptr(parents), _current_stream()))
    return q_out


def stack_attn_decode_batch(q, cache: KVCache, lengths, scale: float, out=None, gate=None,
                            prefix: Optional[KVCache] = None, prefix_len: Optional[int] = None, parents=None,
                            workspace=None, stream=None):
    """out bf16 [rows, hq * d] = softmax(scale q K^T) V (times sigmoid(gate)), token t of
    sequence b attending to the first prefix_len rows of `prefix` (a cache of one sequence that
    all share; default: all of it) and to rows 0 .. lengths[b] + t of its own cache, or its
    path with parents.  workspace: a uint8 tensor of stack_attn_decode_batch_workspace_bytes(),
    allocated for the call when not given; calls that may overlap, captured graphs included,
    need one each."""
    import torch
    ctx = _elsewhere(cache.device, stream)
    if ctx is not None:
        with ctx:
            return stack_attn_decode_batch(q, cache, lengths, scale, out, gate, prefix, prefix_len, parents, workspace)
    dev, d = cache.device, cache.head_dim
    rows, width = q.shape
    T = _block_tokens("q", rows, cache)
    _rows_bf16("q", q, dev)
    hq = width // d
    if hq * d != width:
        raise ValueError(f"q rows of {width} elements are no whole number of heads of {d}")
    if gate is not None:
        _rows_bf16("gate", gate, dev, width)
        if gate.shape[0] != rows:
            raise ValueError(f"gate of {gate.shape[0]} rows for {rows}")
    _ints("lengths", lengths, dev, (cache.sequences,))
    if parents is not None:
        _ints("parents", parents, dev, (cache.sequences, T))
    if out is None:
        out = q.new_empty((rows, width))
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (rows, width) or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out: contiguous bf16 {(rows, width)} on {dev} is expected")
    if prefix is not None and prefix.device != dev:
        raise ValueError(f"the prefix is on {prefix.device}, the cache on {dev}")
    if prefix_len is None:
        prefix_len = prefix.max_len if prefix is not None else 0
    if workspace is None:
        workspace = torch.empty(stack_attn_decode_batch_workspace_bytes(cache, prefix_len, T, hq), dtype=torch.uint8,
                                device=dev)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace: a contiguous tensor on {dev} is expected")
    check(lib.dflash_stack_attn_decode_batch(
        _ptr(q), q.stride(0), _ptr(gate), 0 if gate is None else gate.stride(0), cache.ref, _ptr(lengths),
        None if prefix is None else prefix.ref, prefix_len, _ptr(out), T, hq, scale, _ptr(parents),
        _ptr(workspace), workspace.numel() * workspace.element_size(), _current_stream()))
    return out


def stack_attn_decode_batch_workspace_bytes(cache: KVCache, prefix_len: int, tokens: int, hq: int) -> int:
    return int(lib.dflash_stack_attn_decode_batch_workspace_bytes(cache.ref, prefix_len, tokens, hq))


def stack_kv_read(cache: KVCache, rows: int, starts=None, k=None, v=None, stream=None):
    """Cache rows starts[b] .. starts[b] + rows - 1 of every sequence (starts int32 [sequences]
    on the device; None: from row 0) as bf16 k, v [sequences, kv_heads, rows, head_dim]."""
    ctx = _elsewhere(cache.device, stream)
    if ctx is not None:
        with ctx:
            return stack_kv_read(cache, rows, starts, k, v)
    shape = (cache.sequences, cache.kv_heads, rows, cache.head_dim)
    if starts is not None:
        _ints("starts", starts, cache.device, (cache.sequences,))
    _cache_rows([t for t in (k, v) if t is not None], shape, cache.device)
    bf16 = cache.k[0 if cache.bits == 16 else 1]
    k = bf16.new_empty(shape) if k is None else k
    v = bf16.new_empty(shape) if v is None else v
    check(lib.dflash_stack_kv_read(cache.ref, _ptr(starts), rows, _ptr(k), _ptr(v), _current_stream()))
    return k, v


def _cache_rows(tensors, shape, device):
    import torch
    for t in tensors:
        if t.dtype != torch.bfloat16 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
            raise ValueError(f"cache rows: contiguous bf16 {shape} on {device} are expected, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")


def stack_kv_write(cache: KVCache, k, v, starts=None, stream=None):
    """Rows k, v (bf16 [sequences, kv_heads, rows, head_dim], already normalised and rotated)
    into the cache in its format, from row starts[b] (None: 0) on."""
    ctx = _elsewhere(cache.device, stream)
    if ctx is not None:
        with ctx:
            return stack_kv_write(cache, k, v, starts)
    _cache_rows((k, v), (cache.sequences, cache.kv_heads, k.shape[2], cache.head_dim), cache.device)
    if starts is not None:
        _ints("starts", starts, cache.device, (cache.sequences,))
    check(lib.dflash_stack_kv_write(cache.ref, _ptr(starts), k.shape[2], _ptr(k), _ptr(v), _current_stream()))


def stack_kv_compact_batch(cache: KVCache, lengths, rows, counts, stream=None):
    """After a tree round: cache rows lengths[b] + rows[b, i] -> lengths[b] + i for i < counts[b]
    (int32 on the device: rows [sequences, <= 32], lengths and counts [sequences])."""
    ctx = _elsewhere(cache.device, stream)
    if ctx is not None:
        with ctx:
            return stack_kv_compact_batch(cache, lengths, rows, counts)
    _ints("lengths", lengths, cache.device, (cache.sequences,))
    _ints("counts", counts, cache.device, (cache.sequences,))
    _ints("rows", rows, cache.device, (cache.sequences, rows.shape[-1]))
    check(lib.dflash_stack_kv_compact_batch(cache.ref, _ptr(lengths), _ptr(rows), _ptr(counts), rows.shape[1], _current_stream()))


LOGITS_BF16, LOGITS_FP32 = 0, 1


def logprobs(logits, tokens=None, top: int = 0, stream=None) -> dict:
    """Log probabilities of rows of logits (bf16 or fp32 [rows, vocab], adjacent elements):
    {"logprobs": fp32 [rows, n] at tokens (int32 [rows, n]; 0 for a negative token, NaN for one
    past the vocabulary), "entropy": fp32 [rows], "top_ids": int32 [rows, top], "top_logprobs":
    fp32 [rows, top], the most likely first, the lower id first among equals}."""
    import torch
    ctx = _elsewhere(logits.device, stream)
    if ctx is not None:
        with ctx:
            return logprobs(logits, tokens, top)
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32) or logits.stride(1) != 1:
        raise ValueError(f"logits: bf16 or fp32 [rows, vocab] with adjacent elements are expected, got {logits.dtype} "
                         f"{tuple(logits.shape)} with strides {logits.stride()}")
    rows, vocab = logits.shape
    dev, n = logits.device, 0
    if tokens is not None:
        n = tokens.shape[1] if tokens.dim() == 2 else -1
        _ints("tokens", tokens, dev, (rows, n))
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    logp, best = entropy.new_empty((rows, n)), entropy.new_empty((rows, top))
    ids = torch.empty((rows, top), dtype=torch.int32, device=dev) if tokens is None else tokens.new_empty((rows, top))
    check(lib.dflash_logprobs(_ptr(logits), LOGITS_BF16 if logits.dtype == torch.bfloat16 else LOGITS_FP32,
                              logits.stride(0) if rows > 1 else vocab, rows, vocab, _ptr(tokens), n, top, _ptr(logp),
                              _ptr(entropy), _ptr(ids), _ptr(best), _current_stream()))
    return {"logprobs": logp, "entropy": entropy, "top_ids": ids, "top_logprobs": best}


# ----------------------------------------------------------------------------- the verify stack object

class QWeight(ctypes.Structure):
    """dflash_qweight (include/dflash_stack.h)."""
    _fields_ = [("w", _vp), ("scales", _vp), ("biases", _vp), ("N", _i), ("K", _i)]


class StackLayer(ctypes.Structure):
    """dflash_stack_layer."""
    _fields_ = [("attention", _i), ("ln", _vp), ("post_ln", _vp), ("in_proj", QWeight), ("out_proj", QWeight),
                ("conv", _vp), ("a_log", _vp), ("dt_bias", _vp), ("gdn_norm", _vp), ("snapshot", _vp),
                ("window", _vp), ("qkv", QWeight), ("o_proj", QWeight), ("q_norm", _vp), ("k_norm", _vp),
                ("cache_k", _vp), ("cache_v", _vp), ("gate_up", QWeight), ("down", QWeight)]


class StackDesc(ctypes.Structure):
    """dflash_stack_desc."""
    _fields_ = [("layers", _i), ("hidden", _i), ("block", _i), ("gdn_heads", _i), ("gdn_key_heads", _i),
                ("gdn_dk", _i), ("gdn_dv", _i), ("conv_kernel", _i), ("attn_heads", _i), ("kv_heads", _i),
                ("head_dim", _i), ("rotary_dim", _i), ("max_len", _i), ("rope_theta", _f), ("eps", _f),
                ("group", _i), ("bits", _i), ("rank", _i), ("world", _i), ("vocab0", _i),
                ("layer", ctypes.POINTER(StackLayer)), ("final_norm", _vp), ("lm_head", QWeight),
                ("exchange", _vp), ("key_exchange", _vp)]


def _qweight(q) -> QWeight:
    return QWeight(_ptr(q.w), _ptr(q.scales), _ptr(q.biases), q.N, q.K) if q is not None else QWeight()


class CStack:
    """dflash_stack: the verify stack driven by the library alone (include/dflash_stack.h),
    built over the shard weights and state of a verify_stack.VerifyStack-shaped shard (the
    dicts of build_rank_weights / build_rank_state) — the same buffers, referenced.  The
    exchanges (world > 1) are PeerExchange objects already connected to every rank."""

    def __init__(self, cfg, plan, weights: dict, state: dict, context: int, exchange=None, key_exchange=None):
        p, w = plan, weights
        layers = []
        for L, S in zip(w["layers"], state["layers"]):
            if L["kind"] == "gdn":
                layers.append(StackLayer(0, _ptr(L["ln"]), _ptr(L["post_ln"]), _qweight(L["in_proj"]),
                                         _qweight(L["out_proj"]), _ptr(L["conv"]), _ptr(L["a_log"]),
                                         _ptr(L["dt_bias"]), _ptr(L["gdn_norm"]), _ptr(S["snapshot"]),
                                         _ptr(S["window"]), QWeight(), QWeight(), None, None, None, None,
                                         _qweight(L["gate_up"]), _qweight(L["down"])))
            else:
                layers.append(StackLayer(1, _ptr(L["ln"]), _ptr(L["post_ln"]), QWeight(), QWeight(), None, None,
                                         None, None, None, None, _qweight(L["qkv"]), _qweight(L["o_proj"]),
                                         _ptr(L["q_norm"]), _ptr(L["k_norm"]), _ptr(S["cache_k"]),
                                         _ptr(S["cache_v"]), _qweight(L["gate_up"]), _qweight(L["down"])))
        self._layers = (StackLayer * len(layers))(*layers)
        self._keep = (weights, state, exchange, key_exchange)  # referenced, not copied: keep alive
        max_len = next((S["cache_k"].shape[1] for S in state["layers"] if "cache_k" in S), context + cfg.block)
        self.desc = StackDesc(
            cfg.layers, cfg.hidden, cfg.block, p.gdn_heads, p.gdn_key_heads or p.gdn_heads, cfg.gdn_dk, cfg.gdn_dv,
            cfg.conv_kernel, p.attn_heads, p.kv_heads, cfg.head_dim, cfg.rotary_dim, max_len, cfg.rope_theta,
            cfg.eps, cfg.group, cfg.bits, p.rank, p.world, p.vocab0, self._layers, _ptr(w["final_norm"]),
            _qweight(w["lm_head"]), ctypes.cast(exchange.bases, _vp) if exchange is not None else None,
            ctypes.cast(key_exchange.bases, _vp) if key_exchange is not None else None)
        h = _vp()
        check(lib.dflash_stack_create(ctypes.byref(self.desc), int(context), ctypes.byref(h)))
        self.handle = h

    def forward(self, hidden, out=None, stream=None):
        check(lib.dflash_stack_forward(self.handle, _ptr(hidden), _ptr(out), _stream(stream)))
        return out

    def output_ptr(self) -> int:
        return lib.dflash_stack_output(self.handle)

    def verify(self, hidden, proposals, tokens, accepted, stream=None):
        check(lib.dflash_stack_verify(self.handle, _ptr(hidden), _ptr(proposals), _ptr(tokens), _ptr(accepted),
                                      _stream(stream)))
        return tokens, accepted

    def commit(self, keep: int, stream=None):
        check(lib.dflash_stack_commit(self.handle, None, int(keep), _stream(stream)))

    def advance(self, n: int):
        check(lib.dflash_stack_advance(self.handle, int(n)))

    @property
    def context(self) -> int:
        return int(lib.dflash_stack_context(self.handle))

    def close(self):
        if self.handle:
            lib.dflash_stack_destroy(self.handle)
            self.handle = None
