"""ctypes binding of libmtcuda.so, the C ABI declared in include/mtcuda.h.

This is the binding a Python caller of the B200 backend uses (and what the
GPU parity tests call through).  Operands are `View`s: a flat storage tensor
plus shape, strides and offset in elements, i.e. the reference's
`Materialization{Buffer, Layout}` (src/tensor/storage/materialization.hpp:11-22).
Errors come back as the exception type the reference would throw for the same
condition (std::invalid_argument -> ValueError, std::out_of_range -> IndexError,
std::overflow_error -> OverflowError, std::runtime_error / logic_error ->
RuntimeError).

Loading fails loudly: there is no fallback path when the library is missing.
"""
from __future__ import annotations

import ctypes
import os
import struct
from dataclasses import dataclass, field
from pathlib import Path
from typing import Sequence

MAX_RANK = 8

OK, ERR_INVALID_ARGUMENT, ERR_OUT_OF_RANGE, ERR_RUNTIME, ERR_LOGIC, ERR_OVERFLOW, ERR_UNSUPPORTED = range(7)
FLOAT32, INT64 = 0, 1

# operation codes (reference PrimitiveId values; 0x..80+ are additions)
ABS, SIGN, NEGATE, EXP, LOG, SQRT, TANH, SIGMOID = range(0x0101, 0x0109)
RELU = 0x0180
ADD, SUBTRACT, MULTIPLY, DIVIDE, LOGADDEXP = range(0x0110, 0x0115)
CONST = 0x01F0
SUM, LOGSUMEXP, MAX, ARGMAX = 0x0301, 0x0302, 0x0380, 0x0381
UNARY_OPS = (ABS, SIGN, NEGATE, EXP, LOG, SQRT, TANH, SIGMOID, RELU)
BINARY_OPS = (ADD, SUBTRACT, MULTIPLY, DIVIDE, LOGADDEXP)

NO_TOKEN = -(1 << 63)  # padding_token / ignore_target that excludes nothing

GEMM_AUTO, GEMM_SIMT, GEMM_3XTF32, GEMM_SIMT_FFMA = 0, 1, 2, 3

LIB_DIR = Path(__file__).resolve().parent / "lib"


class Desc(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("offset", ctypes.c_int64),
        ("capacity", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("rank", ctypes.c_int32),
        ("shape", ctypes.c_int64 * MAX_RANK),
        ("strides", ctypes.c_int64 * MAX_RANK),
    ]


# mtc_desc by rank: the unused extents and strides are padding (zeros)
_DESC = [struct.Struct(f"@Pqqii{r}q{8 * (MAX_RANK - r)}x{r}q{8 * (MAX_RANK - r)}x") for r in range(MAX_RANK + 1)]
_PACK = [s.pack for s in _DESC]
assert all(s.size == ctypes.sizeof(Desc) for s in _DESC)


_DTYPES: dict = {}  # torch dtype -> (code, binary logarithm of its size)


def _dtypes() -> dict:
    if not _DTYPES:
        import torch

        _DTYPES.update({torch.float32: (FLOAT32, 2), torch.int64: (INT64, 3)})
    return _DTYPES


class Instr(ctypes.Structure):
    _fields_ = [
        ("op", ctypes.c_int32),
        ("dst", ctypes.c_int16),
        ("a", ctypes.c_int16),
        ("b", ctypes.c_int16),
        ("pad", ctypes.c_int16),
        ("imm", ctypes.c_float),
    ]


def make_desc(ptr: int, capacity: int, dtype: int, shape: Sequence[int], strides: Sequence[int], offset: int) -> Desc:
    if len(shape) != len(strides) or len(shape) > MAX_RANK:
        raise ValueError("shape/strides rank mismatch or rank > 8")
    d = Desc()
    d.data = ptr
    d.offset = int(offset)
    d.capacity = int(capacity)
    d.dtype = int(dtype)
    d.rank = len(shape)
    for i, (e, s) in enumerate(zip(shape, strides)):
        d.shape[i] = int(e)
        d.strides[i] = int(s)
    return d


def contiguous_strides(shape: Sequence[int]) -> list[int]:
    """Layout::contiguous (src/tensor/storage/layout.cpp:23-48): extent-0/1 axes do not grow the stride."""
    strides = [1] * len(shape)
    run = 1
    for i in range(len(shape) - 1, -1, -1):
        strides[i] = run
        if shape[i] >= 2:
            run *= shape[i]
    return strides


def _flat(memory, dtype):
    """A storage as a flat tensor."""
    import torch

    return torch.empty(0, dtype=dtype, device=memory.device).set_(memory)


class _OfTensor:
    """What a view made of a tensor was made of, beside its fields."""

    __slots__ = ("_of",)


@dataclass
class View(_OfTensor):
    """A strided view of a flat storage tensor (torch tensor, on any device)."""

    storage: "object"  # torch.Tensor, 1-D
    shape: tuple
    strides: tuple
    offset: int = field(default_factory=int)

    @staticmethod
    def of(t) -> "View":
        """View of an existing torch tensor as it is now (shares its storage)."""
        memory, dtype, shape = t.untyped_storage(), t.dtype, t.shape
        rank = len(shape)
        code = (_DTYPES or _dtypes()).get(dtype)
        if code is None or rank > MAX_RANK:
            return View(_flat(memory, dtype), tuple(shape), t.stride(), t.storage_offset())
        # The descriptor is packed at once, and the fields and the flat tensor are made when they
        # are asked for: that one tensor costs as much as a small call's launch.
        ptr = memory.data_ptr()
        v = _new_view(View)
        _set_of(v, (ptr, memory, _PACK[rank](ptr, t.storage_offset(), memory.nbytes() >> code[1], code[0], rank, *shape,
                                             *t.stride()), dtype, rank))
        return v

    def __getattr__(self, name):
        if name == "_of":
            return None
        of = self._of
        if of is None or name not in ("storage", "shape", "strides", "offset"):
            raise AttributeError(f"{type(self).__name__!r} object has no attribute {name!r}")
        _, memory, packed, dtype, rank = of
        fields = self.__dict__
        if name == "storage":
            fields["storage"] = _flat(memory, dtype)
        else:
            _, fields["offset"], _, _, _, *axes = _DESC[rank].unpack(packed)
            fields["shape"], fields["strides"] = tuple(axes[:rank]), tuple(axes[rank:])
        return fields[name]

    def __setattr__(self, name, value):
        if self._of is not None:
            self.storage, self.shape  # the fields that are not set stay what the view was made with
            _set_of(self, None)
        object.__setattr__(self, name, value)

    @staticmethod
    def contiguous(storage, shape, offset: int = 0) -> "View":
        return View(storage, tuple(shape), tuple(contiguous_strides(shape)), offset)

    def desc(self) -> Desc:
        import torch

        dt = INT64 if self.storage.dtype == torch.int64 else FLOAT32
        return make_desc(self.storage.data_ptr(), self.storage.numel(), dt, self.shape, self.strides, self.offset)

    def packed(self) -> bytes:
        """The view's descriptor as the bytes of an mtc_desc, in one pack: a call of small
        tensors costs what its descriptors do.  Float32 and Int64 alone."""
        of = self._of
        if of is not None and of[1].data_ptr() == of[0]:  # (a storage that was resized since lies elsewhere)
            return of[2]
        storage = self.storage
        rank = len(self.shape)
        if rank != len(self.strides) or rank > MAX_RANK:
            raise ValueError("shape/strides rank mismatch or rank > 8")
        code = _dtypes().get(storage.dtype)
        if code is None:
            raise ValueError(f"{storage.dtype} operands are not supported: Float32 or Int64")
        return _PACK[rank](storage.data_ptr(), self.offset, storage.numel(), code[0], rank, *self.shape, *self.strides)

    def tensor(self):
        """The same view as a torch tensor (for zero/positive strides)."""
        return self.storage.as_strided(self.shape, self.strides, self.offset)


_new_view, _set_of = object.__new__, _OfTensor._of.__set__


class MtcError(RuntimeError):
    pass


_lib = None


def lib():
    global _lib
    if _lib is not None:
        return _lib
    path = LIB_DIR / "libmtcuda.so"
    try:  # load PyTorch first so its CUDA runtime / NCCL are the process-wide copies
        import torch  # noqa: F401
    except ImportError:
        pass
    if not path.exists():
        raise MtcError(f"libmtcuda.so is not built ({path}); run __graft_entry__.build()")
    _lib = ctypes.CDLL(str(path), mode=os.RTLD_GLOBAL if hasattr(os, "RTLD_GLOBAL") else 0)
    _declare(_lib)
    return _lib


def _declare(L):
    P = ctypes.POINTER
    c_int, c_i32, c_i64, c_f, c_vp, c_sz = ctypes.c_int, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t
    sig = {
        "mtc_last_error": ([], ctypes.c_char_p),
        "mtc_version": ([], ctypes.c_char_p),
        "mtc_device_count": ([P(c_int)], c_int),
        "mtc_device_sm_count": ([c_int, P(c_int)], c_int),
        "mtc_device_stream": ([c_int, P(c_vp)], c_int),
        "mtc_set_device": ([c_int], c_int),
        "mtc_alloc": ([c_int, c_sz, c_vp, P(c_vp)], c_int),
        "mtc_free": ([c_int, c_vp, c_vp], c_int),
        "mtc_copy_from_host": ([c_int, c_vp, c_vp, c_sz, c_vp], c_int),
        "mtc_copy_to_host": ([c_int, c_vp, c_vp, c_sz, c_vp], c_int),
        "mtc_stream_synchronize": ([c_vp], c_int),
        "mtc_pool_stats": ([c_int, P(ctypes.c_uint64), P(ctypes.c_uint64)], c_int),
        "mtc_pool_trim": ([c_int], c_int),
        "mtc_pool_take": ([c_int, c_vp, c_sz, c_vp], c_int),
        "mtc_stream_create": ([c_int, P(c_vp)], c_int),
        "mtc_stream_destroy": ([c_int, c_vp], c_int),
        "mtc_event_create": ([c_int, P(c_vp)], c_int),
        "mtc_event_destroy": ([c_int, c_vp], c_int),
        "mtc_event_record": ([c_vp, c_vp], c_int),
        "mtc_stream_wait_event": ([c_vp, c_vp], c_int),
        "mtc_event_create_timed": ([c_int, P(c_vp)], c_int),
        "mtc_event_elapsed": ([c_vp, c_vp, P(c_f)], c_int),
        "mtc_pool_protect": ([c_int, c_vp, c_i32], c_int),
        "mtc_pool_take_many": ([c_int, P(c_vp), P(c_sz), c_i32, c_vp, P(c_i32)], c_int),
        "mtc_capture_begin": ([c_int, c_vp], c_int),
        "mtc_capture_end": ([c_int, P(c_vp)], c_int),
        "mtc_capture_fused_count": ([P(c_i32)], c_int),
        "mtc_graph_launch": ([c_vp], c_int),
        "mtc_graph_set_constants": ([c_vp, c_i32, P(c_f), c_i32], c_int),
        "mtc_graph_launches": ([c_vp, P(ctypes.c_uint64)], c_int),
        "mtc_graph_destroy": ([c_vp], c_int),
        "mtc_check_device_errors": ([c_int, c_vp, P(c_i64)], c_int),
        "mtc_watch_device_errors": ([c_int, c_vp], c_int),
        "mtc_poll_device_errors": ([c_int, c_int, P(ctypes.c_int64)], c_int),
        "mtc_selftest_bounded_wait": ([c_i64, c_vp], c_int),
        "mtc_unary": ([c_i32, P(Desc), P(Desc), c_vp], c_int),
        "mtc_binary": ([c_i32, P(Desc), P(Desc), P(Desc), c_vp], c_int),
        "mtc_fused": ([P(Instr), c_i32, P(Desc), c_i32, P(c_i32), P(Desc), c_i32, c_vp], c_int),
        "mtc_copy": ([P(Desc), P(Desc), c_vp], c_int),
        "mtc_concat": ([P(Desc), c_i32, c_i64, P(Desc), c_vp], c_int),
        "mtc_index_scatter": ([P(Desc), P(Desc), P(Desc), c_vp], c_int),
        "mtc_gather": ([P(Desc), P(Desc), c_i64, P(Desc), c_vp], c_int),
        "mtc_gather_scatter_add": ([P(Desc), P(Desc), c_i64, P(Desc), c_vp], c_int),
        "mtc_gather_scatter_add_into": ([P(Desc), P(Desc), c_i64, P(Desc), c_vp], c_int),
        # descriptors as untyped pointers: the packed bytes of a view, or byref(Desc)
        "mtc_embedding": ([c_vp, c_vp, c_f, c_i64, c_vp, c_vp], c_int),
        "mtc_embedding_grad": ([c_vp, c_vp, c_f, c_i64, c_i32, c_vp, c_vp], c_int),
        "mtc_linear_cross_entropy": ([c_vp] * 4 + [c_i64, c_vp, c_vp, c_vp], c_int),
        "mtc_linear_cross_entropy_grad": ([c_vp] * 4 + [c_i64] + [c_vp] * 7, c_int),
        "mtc_token_log_probs": ([c_vp, c_vp, c_f, c_i64] + [c_vp] * 6, c_int),
        "mtc_token_log_probs_grad": ([c_vp, c_vp, c_f, c_i64] + [c_vp] * 4, c_int),
        "mtc_global_norm": ([c_vp, c_i32, c_vp, c_vp], c_int),
        "mtc_clip_global_norm": ([c_vp, c_i32, c_f, c_vp, c_vp, c_vp], c_int),
        "mtc_orthogonalize": ([c_vp, c_i32, c_vp, c_i32, c_f, c_vp, c_vp], c_int),
        "mtc_reduce": ([c_i32, P(Desc), P(c_i64), c_i32, P(Desc), c_vp], c_int),
        "mtc_log_softmax": ([P(Desc), c_i64, P(Desc), c_vp], c_int),
        "mtc_matmul": ([P(Desc), P(Desc), P(Desc), c_i32, c_vp], c_int),
        "mtc_matmul_3xtf32_static": ([P(Desc), P(Desc), P(Desc), c_vp], c_int),
        "mtc_fill": ([P(Desc), c_vp, c_vp], c_int),
        "mtc_uniform": ([P(Desc), c_f, c_f, ctypes.c_uint64, ctypes.c_uint64, c_vp], c_int),
        "mtc_normal": ([P(Desc), c_f, c_f, ctypes.c_uint64, ctypes.c_uint64, c_vp], c_int),
        "mtc_launch_count": ([P(ctypes.c_uint64)], c_int),
        "mtc_profile_enable": ([c_int], c_int),
        "mtc_profile_gemm": ([P(ctypes.c_uint64), P(ctypes.c_double), P(ctypes.c_double), c_int], c_int),
        "mtc_gemm_path_counts": ([P(ctypes.c_uint64), P(ctypes.c_uint64)], c_int),
        "mtc_comm_unique_id": ([c_vp, c_sz], c_int),
        "mtc_comm_init": ([c_int, c_int, c_int, c_vp, c_sz, P(c_vp)], c_int),
        "mtc_comm_allreduce_f32": ([c_vp, P(c_vp), P(c_sz), c_i32, c_f, c_vp], c_int),
        "mtc_comm_allreduce_f32_async": ([c_vp, P(c_vp), P(c_sz), c_i32, c_f, c_vp], c_int),
        "mtc_comm_wait": ([c_vp, c_vp], c_int),
        "mtc_comm_destroy": ([c_vp], c_int),
    }
    for name, (args, res) in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = res


EXPORTED = (
    "mtc_last_error", "mtc_version", "mtc_device_count", "mtc_device_sm_count", "mtc_set_device", "mtc_device_stream", "mtc_alloc",
    "mtc_free", "mtc_copy_from_host", "mtc_copy_to_host", "mtc_stream_synchronize", "mtc_pool_stats", "mtc_pool_trim",
    "mtc_stream_create", "mtc_stream_destroy", "mtc_event_create", "mtc_event_destroy", "mtc_event_record",
    "mtc_stream_wait_event", "mtc_event_create_timed", "mtc_event_elapsed", "mtc_pool_take", "mtc_pool_take_many", "mtc_pool_protect", "mtc_capture_begin", "mtc_capture_end", "mtc_capture_fused_count", "mtc_graph_launch",
    "mtc_graph_set_constants", "mtc_graph_launches", "mtc_graph_destroy",
    "mtc_check_device_errors", "mtc_watch_device_errors", "mtc_poll_device_errors", "mtc_selftest_bounded_wait", "mtc_unary", "mtc_binary", "mtc_fused", "mtc_copy", "mtc_concat", "mtc_index_scatter",
    "mtc_gather", "mtc_gather_scatter_add", "mtc_gather_scatter_add_into", "mtc_embedding", "mtc_embedding_grad", "mtc_linear_cross_entropy", "mtc_linear_cross_entropy_grad", "mtc_token_log_probs", "mtc_token_log_probs_grad", "mtc_global_norm", "mtc_clip_global_norm", "mtc_orthogonalize", "mtc_reduce", "mtc_log_softmax", "mtc_matmul", "mtc_fill", "mtc_uniform",
    "mtc_normal", "mtc_launch_count", "mtc_profile_enable", "mtc_profile_gemm", "mtc_gemm_path_counts", "mtc_comm_unique_id", "mtc_comm_init", "mtc_comm_allreduce_f32", "mtc_comm_allreduce_f32_async", "mtc_comm_wait", "mtc_comm_destroy",
)


def check(rc: int, what: str = "") -> None:
    if rc == OK:
        return
    msg = lib().mtc_last_error().decode(errors="replace")
    text = f"{what}: {msg}" if what else msg
    if rc == ERR_INVALID_ARGUMENT:
        raise ValueError(text)
    if rc == ERR_OUT_OF_RANGE:
        raise IndexError(text)
    if rc == ERR_OVERFLOW:
        raise OverflowError(text)
    raise MtcError(f"[code {rc}] {text}")


def _stream(stream):
    if stream is None:
        import torch

        # the handle alone, where this torch has a function for it: a Stream object costs more
        # than a small call's launch
        handle = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if handle is None:
            return torch.cuda.current_stream().cuda_stream
        return handle(torch.cuda.current_device())
    return ctypes.c_void_p(int(stream))


# ------------------------------------------------------------------ wrappers --
# Every kernel wrapper takes `prepare=True` to return a zero-argument callable
# with its ctypes arguments converted once: repeated calls then cost one ctypes
# dispatch, so back-to-back launches keep the GPU busy in timing loops.

_FUNCTIONS: dict = {}


def _run(name: str, args: tuple, what: str, prepare: bool):
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(lib(), name)
    if prepare:
        def call() -> None:
            check(fn(*args), what)
        return call
    rc = fn(*args)
    if rc != OK:
        check(rc, what)
    return None


def unary(op: int, x: View, out: View, stream=None, prepare: bool = False):
    return _run("mtc_unary", (op, ctypes.byref(x.desc()), ctypes.byref(out.desc()), _stream(stream)), "unary", prepare)


def binary(op: int, a: View, b: View, out: View, stream=None, prepare: bool = False):
    return _run("mtc_binary", (op, ctypes.byref(a.desc()), ctypes.byref(b.desc()), ctypes.byref(out.desc()),
                               _stream(stream)), "binary", prepare)


def fused(program: Sequence[tuple], inputs: Sequence[View], out_regs: Sequence[int], outputs: Sequence[View],
          stream=None, prepare: bool = False):
    """program: (op, dst, a, b, imm) tuples."""
    n = len(program)
    instrs = (Instr * max(n, 1))()
    for i, (op, dst, a, b, imm) in enumerate(program):
        instrs[i].op, instrs[i].dst, instrs[i].a, instrs[i].b, instrs[i].imm = op, dst, a, b, imm
    ins = (Desc * max(len(inputs), 1))(*[v.desc() for v in inputs])
    outs = (Desc * len(outputs))(*[v.desc() for v in outputs])
    regs = (ctypes.c_int32 * len(out_regs))(*out_regs)
    return _run("mtc_fused", (instrs, n, ins, len(inputs), regs, outs, len(outputs), _stream(stream)), "fused",
                prepare)


def copy(src: View, dst: View, stream=None, prepare: bool = False):
    return _run("mtc_copy", (ctypes.byref(src.desc()), ctypes.byref(dst.desc()), _stream(stream)), "copy", prepare)


def concat(inputs: Sequence[View], axis: int, out: View, stream=None, prepare: bool = False):
    arr = (Desc * len(inputs))(*[v.desc() for v in inputs])
    return _run("mtc_concat", (arr, len(inputs), axis, ctypes.byref(out.desc()), _stream(stream)), "concat", prepare)


def index_scatter(x: View, dst_view: View, out: View, stream=None, prepare: bool = False):
    return _run("mtc_index_scatter", (ctypes.byref(x.desc()), ctypes.byref(dst_view.desc()), ctypes.byref(out.desc()),
                                      _stream(stream)), "index_scatter", prepare)


def gather(src: View, idx: View, axis: int, out: View, stream=None, prepare: bool = False):
    return _run("mtc_gather", (ctypes.byref(src.desc()), ctypes.byref(idx.desc()), axis, ctypes.byref(out.desc()),
                               _stream(stream)), "gather", prepare)


def gather_scatter_add(upd: View, idx: View, axis: int, out: View, stream=None, prepare: bool = False):
    return _run("mtc_gather_scatter_add", (ctypes.byref(upd.desc()), ctypes.byref(idx.desc()), axis,
                                           ctypes.byref(out.desc()), _stream(stream)), "gather_scatter_add", prepare)


def _ref(v: View | None):
    return None if v is None else v.packed()


def _packed_all(views: Sequence[View]) -> bytes:
    # (as View.packed does it, without a call for each of many tensors)
    return b"".join([of[2] if (of := v._of) is not None and of[1].data_ptr() == of[0] else v.packed() for v in views])


def _token(t: int | None) -> int:
    return NO_TOKEN if t is None else int(t)


def embedding(table: View, tokens: View, out: View, scale: float = 1.0, padding_token: int | None = None, stream=None,
              prepare: bool = False):
    """out[i.., :] = scale * table[tokens[i..], :]; zeros where the token is `padding_token`."""
    return _run("mtc_embedding", (_ref(table), _ref(tokens), scale, _token(padding_token), _ref(out), _stream(stream)),
                "embedding", prepare)


def embedding_grad(dout: View, tokens: View, dtable: View, scale: float = 1.0, padding_token: int | None = None,
                   accumulate: bool = False, stream=None, prepare: bool = False):
    """dtable[v, :] = scale * the sum of dout over v's positions (added to dtable with `accumulate`)."""
    return _run("mtc_embedding_grad", (_ref(dout), _ref(tokens), scale, _token(padding_token), int(accumulate),
                                       _ref(dtable), _stream(stream)), "embedding_grad", prepare)


def linear_cross_entropy(x: View, weight: View, targets: View, loss: View, bias: View | None = None,
                         lse: View | None = None, ignore_target: int | None = None, stream=None,
                         prepare: bool = False):
    """loss[n] = logsumexp(z[n]) - z[n, targets[n]] with z = x . weight^T + bias, whose logits the caller never holds."""
    return _run("mtc_linear_cross_entropy", (_ref(x), _ref(weight), _ref(bias), _ref(targets), _token(ignore_target),
                                             _ref(loss), _ref(lse), _stream(stream)), "linear_cross_entropy", prepare)


def linear_cross_entropy_grad(x: View, weight: View, targets: View, dloss: View, dx: View | None = None,
                              dweight: View | None = None, bias: View | None = None, dbias: View | None = None,
                              loss: View | None = None, lse: View | None = None, ignore_target: int | None = None,
                              stream=None, prepare: bool = False):
    """linear_cross_entropy with the gradients of sum(dloss * loss) for x, weight and bias."""
    return _run("mtc_linear_cross_entropy_grad",
                (_ref(x), _ref(weight), _ref(bias), _ref(targets), _token(ignore_target), _ref(dloss), _ref(loss),
                 _ref(lse), _ref(dx), _ref(dweight), _ref(dbias), _stream(stream)), "linear_cross_entropy_grad", prepare)


def token_log_probs(logits: View, tokens: View | None = None, log_probs: View | None = None, lse: View | None = None,
                    entropy: View | None = None, top_log_probs: View | None = None, top_tokens: View | None = None,
                    scale: float = 1.0, ignore_token: int | None = None, stream=None, prepare: bool = False):
    """log_probs[i..] = z[i.., tokens[i..]] - logsumexp(z[i..]) with z = scale * logits, the entropy of softmax(z)
    and its likeliest alternatives."""
    return _run("mtc_token_log_probs",
                (_ref(logits), _ref(tokens), scale, _token(ignore_token), _ref(log_probs), _ref(lse), _ref(entropy),
                 _ref(top_log_probs), _ref(top_tokens), _stream(stream)), "token_log_probs", prepare)


def token_log_probs_grad(logits: View, dlogits: View, tokens: View | None = None, dlog_probs: View | None = None,
                         dentropy: View | None = None, scale: float = 1.0, ignore_token: int | None = None,
                         stream=None, prepare: bool = False):
    """dlogits = the gradient of sum(dlog_probs * log_probs) + sum(dentropy * entropy); in place where it is logits."""
    return _run("mtc_token_log_probs_grad",
                (_ref(logits), _ref(tokens), scale, _token(ignore_token), _ref(dlog_probs), _ref(dentropy),
                 _ref(dlogits), _stream(stream)), "token_log_probs_grad", prepare)


def global_norm(tensors: Sequence[View], norm: View, stream=None, prepare: bool = False):
    """norm = sqrt of the sum of squares of all elements of all tensors."""
    arr = _packed_all(tensors)
    return _run("mtc_global_norm", (arr, len(tensors), _ref(norm), _stream(stream)), "global_norm", prepare)


def clip_global_norm(tensors: Sequence[View], max_norm: float, norm: View | None = None,
                     outs: Sequence[View] | None = None, stream=None, prepare: bool = False):
    """Scales the tensors by max_norm / norm where their global norm exceeds max_norm; into `outs`, or in place."""
    arr = _packed_all(tensors)
    if outs is not None and len(outs) != len(tensors):
        raise ValueError(f"{len(outs)} outputs for {len(tensors)} tensors")
    to = arr if outs is None else _packed_all(outs)
    return _run("mtc_clip_global_norm", (arr, len(tensors), max_norm, to, _ref(norm), _stream(stream)),
                "clip_global_norm", prepare)


# (a, b, c) of a step that takes singular values of [0.01, 1] to about [0.7, 1.2] in five
QUINTIC = (3.4445, -4.7750, 2.0315)


def orthogonalize(tensors: Sequence[View], outs: Sequence[View] | None = None,
                  coefficients: Sequence[Sequence[float]] = (QUINTIC,) * 5, eps: float = 1e-7, stream=None,
                  prepare: bool = False):
    """X = T / (|T| + eps), then X <- a X + (b S + c S^2) X with S = X X^T for each (a, b, c), of every matrix T of
    the tensors (their last two axes, on the shorter side); into `outs`, or in place."""
    arr = _packed_all(tensors)
    if outs is not None and len(outs) != len(tensors):
        raise ValueError(f"{len(outs)} outputs for {len(tensors)} tensors")
    to = arr if outs is None else _packed_all(outs)
    flat = [float(v) for step in coefficients for v in step]
    if any(len(step) != 3 for step in coefficients):
        raise ValueError("coefficients are not of three numbers a step")
    table = (ctypes.c_float * max(len(flat), 1))(*flat)
    return _run("mtc_orthogonalize", (arr, len(tensors), table, len(coefficients), eps, to, _stream(stream)),
                "orthogonalize", prepare)


def reduce(op: int, x: View, axes: Sequence[int], out: View, stream=None, prepare: bool = False):
    ax = (ctypes.c_int64 * max(len(axes), 1))(*axes)
    return _run("mtc_reduce", (op, ctypes.byref(x.desc()), ax, len(axes), ctypes.byref(out.desc()), _stream(stream)),
                "reduce", prepare)


def log_softmax(x: View, axis: int, out: View, stream=None, prepare: bool = False):
    return _run("mtc_log_softmax", (ctypes.byref(x.desc()), axis, ctypes.byref(out.desc()), _stream(stream)),
                "log_softmax", prepare)


def matmul(a: View, b: View, out: View, algo: int = GEMM_AUTO, stream=None, prepare: bool = False):
    return _run("mtc_matmul", (ctypes.byref(a.desc()), ctypes.byref(b.desc()), ctypes.byref(out.desc()), algo,
                               _stream(stream)), "matmul", prepare)


def fill(out: View, value, stream=None) -> None:
    import torch

    if out.storage.dtype == torch.int64:
        v = ctypes.c_int64(int(value))
    else:
        v = ctypes.c_float(float(value))
    check(lib().mtc_fill(ctypes.byref(out.desc()), ctypes.byref(v), _stream(stream)), "fill")


def uniform(out: View, low: float, high: float, key: tuple, stream=None) -> None:
    check(lib().mtc_uniform(ctypes.byref(out.desc()), low, high, key[0], key[1], _stream(stream)), "uniform")


def normal(out: View, mean: float, std: float, key: tuple, stream=None) -> None:
    check(lib().mtc_normal(ctypes.byref(out.desc()), mean, std, key[0], key[1], _stream(stream)), "normal")


def launch_count() -> int:
    n = ctypes.c_uint64(0)
    check(lib().mtc_launch_count(ctypes.byref(n)))
    return n.value


def profile_enable(on: bool) -> None:
    check(lib().mtc_profile_enable(int(on)))


def profile_gemm(reset: bool = True):
    """(launches, total ms, total FLOPs) of GEMM launches since the last reset."""
    n, ms, fl = ctypes.c_uint64(0), ctypes.c_double(0.0), ctypes.c_double(0.0)
    check(lib().mtc_profile_gemm(ctypes.byref(n), ctypes.byref(ms), ctypes.byref(fl), int(reset)))
    return n.value, ms.value, fl.value


def gemm_path_counts():
    """(tensor-core calls, SIMT calls) of mtc_matmul since the process started."""
    tc, simt = ctypes.c_uint64(0), ctypes.c_uint64(0)
    check(lib().mtc_gemm_path_counts(ctypes.byref(tc), ctypes.byref(simt)))
    return tc.value, simt.value


def check_device_errors(device: int = 0, stream=None) -> None:
    detail = ctypes.c_int64(0)
    check(lib().mtc_check_device_errors(device, _stream(stream), ctypes.byref(detail)), "device error word")
