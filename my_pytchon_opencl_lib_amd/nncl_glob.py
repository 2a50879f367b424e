"""Host-side operator API of the matmul path, mirroring the reference's NnClGlob.

Reference interfaces mirrored (paths relative to the reference repository;
"cs/" = csharp/cstorchcl/cstorchcl/):
  C# NnClGlob (cs/compiler/NnClGlob.cs)        this module
  ------------------------------------------   ---------------------------------------
  Tensor Bmm(Tensor a, Tensor b)      :441     NnClGlob.Bmm(a, b)
  Tensor BmmPermute(a, b, transA, transB):1702 NnClGlob.BmmPermute(a, b, transA, transB)
  Tensor Permute(Tensor x, int[] axes) :382    NnClGlob.Permute(x, axes)
  Tensor LinearForward(x, w, bias)    :1493    NnClGlob.LinearForward(x, w, bias)
  Tensor LinearBiasBackward(g, shape) :1557    NnClGlob.LinearBiasBackward(g, shape)
  Tensor Sum(x, axis, keepDims)       :1595    NnClGlob.Sum(x, axis, keepDims)
  LstmWithWithState gate loop        :1067    NnClGlob.LstmHidGates(x, w, u, bias, hPrev,
                                                                   hOut, workspace, t)
  Python NnClGlob (compiler/nncl_glob.py)
  bmm(A, B)                           :110     NnClGlob.bmm(A, B)
  permute(x, axes)                    :148     NnClGlob.permute(x, axes)
  bmm_backward(grad_output, A, B)     :283     NnClGlob.bmm_backward(grad_output, A, B)

Beyond the reference, for serving in 8 bits: QuantizeRows, NormInt8 (rows of activations in 8
bits, as they are or normed), MatmulInt8, LinearInt8 (layers with int8 weights; an activation, a
gate and a residual in their launch), CacheTables, CacheSlots, CacheRelease, CacheAppend, CacheRead,
CacheAttention (an int8 paged cache, cache.Int8Cache, and the attention that reads it) and Sample
(a token for each row of logits).

Tensors are torch float32 tensors resident on the GPU (torch is only the device-memory and
stream plumbing); every operator enqueues a HIP kernel of libmigemm.so on the current torch
stream through the C ABI. There is no CPU fallback: a CPU tensor or a missing library raises.

Deliberate differences from the reference, each an aliasing or safety fix:
  * every call returns a fresh output tensor; the reference's name-keyed buffer pool makes
    every Bmm output the same "bmm_c" buffer (NnClGlob.cs:460, OpenCLBufferManager.cs:29-40);
  * bmm_backward / BmmOp.Backward use the NT / TN kernels directly instead of
    Permute + Bmm (BmmOp.cs:44-60, nncl_glob.py:300-310) -- same mathematics, no transposed
    copies, and grad_A is no longer overwritten by grad_B;
  * BmmPermute and LinearForward also validate batch / inner sizes, which the reference
    leaves unchecked (an out-of-bounds read there).
"""
import ctypes
import math
import operator
import struct

import torch

from . import _native


class ShapeError(ValueError, AssertionError):
    """Shape / rank / broadcast error raised before any launch. It is an AssertionError for
    callers of the Python reference (which asserts, nncl_glob.py:116-118) and a ValueError
    (the ArgumentException of NnClGlob.cs:443-452) for everyone else."""


def _require(cond, msg):
    if not cond:
        raise ShapeError(msg)


_ptr = torch.Tensor.data_ptr

# The current stream of a device as an integer (torch.cuda.current_stream builds a Stream
# object, 1.9 us; this call 0.1 us).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)

_INT_RANGES = {ctypes.c_int: (-2 ** 31, 2 ** 31 - 1), ctypes.c_int64: (-2 ** 63, 2 ** 63 - 1)}
_entries = {}


def _entry(name):
    """(C function, picker of its integer arguments, their range check) of an entry point."""
    e = _entries.get(name)
    if e is None:
        argtypes = _native.SIGNATURES[name][0][1:]
        ints = [i for i, t in enumerate(argtypes) if t in _INT_RANGES]
        ints.append(ints[-1])  # (itemgetter of a single index would return no tuple)
        # struct packs the integers by their C types and raises on one that does not fit
        pack = struct.Struct("=" + "".join("i" if argtypes[i] is ctypes.c_int else "q"
                                           for i in ints)).pack
        e = _entries[name] = (getattr(_native.load(), name), operator.itemgetter(*ints), pack)
    return e


def _check_ranges(name, args):
    argtypes = _native.SIGNATURES[name][0][1:]
    for i, (t, v) in enumerate(zip(argtypes, args)):
        if t in _INT_RANGES and isinstance(v, int):
            lo, hi = _INT_RANGES[t]
            _require(lo <= v <= hi, f"{name}: argument {i + 1} = {v} does not fit the C "
                                    f"ABI's {'int32' if t is ctypes.c_int else 'int64'}")


def _launch(name, tensors, *args):
    """Calls C-ABI entry `name` on the current stream of the tensors' device, with that
    device current (the library launches on the current HIP device). All tensors of one
    call must live on one device. Integer arguments are range-checked against the C types
    first: ctypes would silently wrap a size or stride of 2^31 or more into a valid-looking
    int32 (the reference's kernels take int sizes and strides, matmul.cl:8-14, 78-87).

    The smallest products take a few microseconds on the GPU, so this path is kept short:
    no message is formatted unless a check fails, the integers are checked in one call, and
    the device is switched only when another one is current (one NnClGlob.BmmPermute call,
    host time: 15.8 -> 8.6 us;
    LstmHidGates, with seven operands, 19.1 -> 7.5)."""
    fn, pick, pack = _entry(name)
    try:
        pack(*pick(args))
    except struct.error:
        _check_ranges(name, args)
    dev = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != dev:
            devices = sorted({str(t.device) for t in tensors})
            raise ShapeError(f"all operands must be on one device (got {devices})")
    if dev == torch.cuda.current_device():
        status = fn(_raw_stream(dev), *args)
    else:
        with torch.cuda.device(dev):
            status = fn(_raw_stream(dev), *args)
    if status:
        _native.check(status)


def _synchronize(t):
    """Waits for the current stream of the tensor's device (the reference's Finish())."""
    dev = t.get_device()
    if dev == torch.cuda.current_device():
        _native.call("migemm_stream_synchronize", _raw_stream(dev))
    else:  # (the null stream is the current device's)
        with torch.cuda.device(dev):
            _native.call("migemm_stream_synchronize", _raw_stream(dev))


def _check_tensor(name, t):
    if isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.is_cuda and \
            t.is_contiguous():
        return
    _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    _require(t.dtype == torch.float32, f"{name} must be float32 (got {t.dtype})")
    _require(t.is_cuda, f"{name} must live on the GPU: the matmul path has no CPU fallback")
    _require(t.is_contiguous(), f"{name} must be contiguous (row-major, as Tensor.cs:283-295)")


# Activations of the 8-bit operators.
_TYPES = {torch.float32: _native.MIGEMM_FLOAT32, torch.bfloat16: _native.MIGEMM_BFLOAT16}


def _check_rows(name, t, dim=None):
    """An activation tensor of the 8-bit operators: float32 or bfloat16, on the GPU. Returns the
    type's code. (Here and below what usually holds is checked in one expression, and a message
    is made only where it does not: a step of a small batch is a few microseconds of GPU work.)"""
    if isinstance(t, torch.Tensor) and t.is_cuda and (dim is None or t.dim() == dim):
        code = _TYPES.get(t.dtype)
        if code is not None:
            return code
    _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    if t.dtype not in _TYPES:
        raise ShapeError(f"{name} must be float32 or bfloat16 (got {t.dtype})")
    _require(t.is_cuda, f"{name} must live on the GPU: there is no CPU fallback")
    raise ShapeError(f"{name} must have {dim} axes (got {list(t.shape)})")


def _row_stride(name, t):
    """Elements between the rows t[i] of a tensor whose rows are contiguous blocks."""
    if t.is_contiguous():
        return t.numel() // t.shape[0] if t.shape[0] else 0
    want = 1
    for n, step in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if n != 1 and step != want:
            raise ShapeError(f"the rows of {name} must be contiguous (strides "
                             f"{list(t.stride())} of {list(t.shape)})")
        want *= n
    if t.shape[0] <= 1:
        return want
    if t.stride(0) < want:
        raise ShapeError(f"the rows of {name} overlap (strides {list(t.stride())} of "
                         f"{list(t.shape)})")
    return t.stride(0)


def _check_typed(name, t, dtype, shape=None, dim=None):
    """A contiguous GPU tensor of one type, and of a shape or a number of axes."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.is_contiguous() and \
            (shape is None or t.shape == shape) and (dim is None or t.dim() == dim):
        return
    _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise ShapeError(f"{name} must be {dtype} (got {t.dtype})")
    _require(t.is_cuda, f"{name} must live on the GPU: there is no CPU fallback")
    if not t.is_contiguous():
        raise ShapeError(f"{name} must be contiguous (strides {list(t.stride())})")
    raise ShapeError(f"{name} must have the shape {list(shape)} (got {list(t.shape)})"
                     if shape is not None else
                     f"{name} must have {dim} axes (got {list(t.shape)})")


_MOST = torch.finfo(torch.float32).max

_ACTIVATIONS = {None: _native.MIGEMM_ACT_NONE, "relu": _native.MIGEMM_ACT_RELU,
                "silu": _native.MIGEMM_ACT_SILU, "gelu": _native.MIGEMM_ACT_GELU,
                "gelu_tanh": _native.MIGEMM_ACT_GELU_TANH}


def _closing(wide, activation, gated):
    """(columns of the output, (activation, gated) as the C entries take them; None for the product
    alone) of a weight of `wide` rows."""
    if activation is None and not gated:
        return wide, None
    if activation not in _ACTIVATIONS:
        names = [a for a in _ACTIVATIONS if a]
        raise ShapeError(f"activation must be None or one of {names} (got {activation!r})")
    if gated and wide % 2:
        raise ShapeError(f"a gated weight must have an even number of rows (got {wide})")
    return wide // 2 if gated else wide, (_ACTIVATIONS[activation], int(bool(gated)))


def _check_residual(t, out):
    """A residual [rows, columns] of the output's type and shape; its rows may lie apart."""
    if _check_rows("residual", t, 2) != _TYPES[out.dtype] or t.shape != out.shape:
        raise ShapeError(f"residual must be {out.dtype} {list(out.shape)} (got {t.dtype} "
                         f"{list(t.shape)})")


def _residual_at(t):
    return (None, 0) if t is None else (_ptr(t), _row_stride("residual", t))


def _check_table(lengths, table):
    """Lengths [requests] and a block table [requests, pages]; returns the table's shape."""
    _check_typed("lengths", lengths, torch.int32, dim=1)
    _check_typed("table", table, torch.int32, dim=2)
    requests, columns = table.shape
    if lengths.shape[0] != requests:
        raise ShapeError(f"table must have {lengths.shape[0]} rows (got {requests})")
    return requests, columns


class NnClGlob:
    """Operator dispatcher of the matmul path (the drop-in for NnClGlob's GEMM ops)."""

    def __init__(self, device=None):
        _native.load()
        self.device = torch.device(device) if device is not None else torch.device("cuda", 0)

    # ------------------------------------------------------------------ C# names
    def Bmm(self, a, b):
        """C[B,M,N] = a[B,M,K] @ b[B|1,K,N]; b with batch 1 is broadcast (stride 0).
        Synchronous, like the reference's Finish() (NnClGlob.cs:498)."""
        _check_tensor("a", a)
        _check_tensor("b", b)
        _require(a.dim() == 3 and b.dim() == 3, "Bmm expects 3-D tensors [Batch, M, K]")
        if not (a.shape[0] == b.shape[0] or b.shape[0] == 1):
            raise ShapeError(f"batch mismatch: {a.shape[0]} and {b.shape[0]}")
        if a.shape[2] != b.shape[1]:
            raise ShapeError(f"inner dimensions differ: K={a.shape[2]} != {b.shape[1]}")
        batch, m, k = a.shape
        n = b.shape[2]
        c = torch.empty((batch, m, n), dtype=torch.float32, device=a.device)
        sB = 0 if b.shape[0] == 1 else k * n
        _launch("migemm_bmm_tiled", (a, b, c), _ptr(a), _ptr(b), _ptr(c), m, k, n, m * k, sB,
                m * n, batch)
        _synchronize(a)
        return c

    def BmmPermute(self, a, b, transA=False, transB=False):
        """C = op(a) @ op(b) with op = transpose of the last two axes when requested
        (NnClGlob.cs:1702-1751). Batch = a.shape[0]; an operand with batch 1 is broadcast.
        Asynchronous on the current stream, like the reference."""
        _check_tensor("a", a)
        _check_tensor("b", b)
        _require(a.dim() == 3 and b.dim() == 3, "BmmPermute expects 3-D tensors")
        batch = a.shape[0]
        m = a.shape[2] if transA else a.shape[1]
        kA = a.shape[1] if transA else a.shape[2]
        kB = b.shape[2] if transB else b.shape[1]
        n = b.shape[1] if transB else b.shape[2]
        if kA != kB:
            raise ShapeError(f"inner dimensions differ: {kA} != {kB}")
        if not (b.shape[0] in (batch, 1)):
            raise ShapeError(f"batch mismatch: {batch} and {b.shape[0]}")
        c = torch.empty((batch, m, n), dtype=torch.float32, device=a.device)
        sA = 0 if a.shape[0] == 1 else a.shape[1] * a.shape[2]
        sB = 0 if b.shape[0] == 1 else b.shape[1] * b.shape[2]
        _launch("migemm_bmm_permute_tiled", (a, b, c), _ptr(a), _ptr(b), _ptr(c), m, kA, n, sA,
                sB, m * n, int(bool(transA)), int(bool(transB)), batch)
        return c

    def Permute(self, x, axes):
        """y = x.permute(axes) materialised (NnClGlob.cs:382-424), up to 10-D."""
        _check_tensor("x", x)
        axes = [int(v) for v in axes]
        _require(len(axes) == x.dim(), "the number of axes must equal the tensor rank")
        if sorted(axes) != list(range(x.dim())):
            raise ShapeError(f"axes {axes} is not a permutation")
        y = torch.empty([x.shape[i] for i in axes], dtype=torch.float32, device=x.device)
        dims = (ctypes.c_int * x.dim())(*x.shape)
        ax = (ctypes.c_int * x.dim())(*axes)
        _launch("migemm_tensor_permute", (x, y), _ptr(x), _ptr(y), dims, ax, x.dim())
        return y

    def LinearForward(self, x, w, bias):
        """Y[B,M,N] = x[B,M,K] @ w[1,K,N] + bias[N], bias added after the k loop
        (NnClGlob.cs:1493-1551, linear.cl:107-143)."""
        _check_tensor("x", x)
        _check_tensor("w", w)
        _check_tensor("bias", bias)
        _require(x.dim() == 3, "LinearForward expects x [Batch, M, K]")
        batch, m, k = x.shape
        n = w.shape[-1]
        if not (w.numel() == k * n and w.shape[-2] == k):
            raise ShapeError(f"w must be [1, {k}, N] (got {list(w.shape)})")
        if bias.numel() != n:
            raise ShapeError(f"bias must have {n} elements (got {bias.numel()})")
        y = torch.empty((batch, m, n), dtype=torch.float32, device=x.device)
        _launch("migemm_linear_forward", (x, w, bias, y), _ptr(x), _ptr(w), _ptr(bias), _ptr(y),
                m, k, n, m * k, m * n, batch)
        return y

    def LinearBiasBackward(self, gradOutput, biasShape):
        """grad_bias[n] = sum over batch and rows of gradOutput (NnClGlob.cs:1557-1584)."""
        _check_tensor("gradOutput", gradOutput)
        n = gradOutput.shape[-1]
        rows = gradOutput.numel() // n
        gb = torch.empty(list(biasShape), dtype=torch.float32, device=gradOutput.device)
        if gb.numel() != n:
            raise ShapeError(f"bias shape {list(biasShape)} does not hold {n} values")
        _launch("migemm_linear_bias_backward", (gradOutput, gb), _ptr(gradOutput), _ptr(gb),
                rows, n)
        return gb

    # ---- LSTM GEMM stages (NnClGlob.Lstm / LstmBackward, cs/compiler/NnClGlob.cs:850-1061).
    # The recurrent kernels between them (lstm_recurrent_forward / _backward) are not part
    # of the matmul path; these are the three GEMM launches of those two methods.
    def LstmGemmXW(self, x, w, bias):
        """XW[T, 4H] = x[B, S, F] (as [T, F]) @ w[F, 4H] + bias[4H]: stage 1 of NnClGlob.Lstm
        (NnClGlob.cs:877-899, lstm_gemm_xw lstm.cl:273-367)."""
        _check_tensor("x", x)
        _check_tensor("w", w)
        _check_tensor("bias", bias)
        f = x.shape[-1]
        t = x.numel() // f
        if not (w.dim() == 2 and w.shape[0] == f):
            raise ShapeError(f"w must be [{f}, 4*hidden] (got {list(w.shape)})")
        g = w.shape[1]
        if bias.numel() != g:
            raise ShapeError(f"bias must have {g} elements (got {bias.numel()})")
        xw = torch.empty((t, g), dtype=torch.float32, device=x.device)
        _launch("migemm_lstm_gemm_xw", (x, w, bias, xw), _ptr(x), _ptr(w), _ptr(bias), _ptr(xw),
                t, f, g)
        return xw

    def LstmRecurrentGates(self, xw, hOut, u, t):
        """The recurrent product of step t inside lstm_recurrent_forward (lstm.cl:80-101,
        enqueued by NnClGlob.Lstm, NnClGlob.cs:912-928), in place on xw [B, S, 4H]:
        xw[:, t] += hOut[:, t-1] @ u (u [H, 4H]); xw[:, t] then holds the step's raw gates
        (the reference's workspace[t, b, :4H], lstm.cl:103-106). A no-op at t = 0."""
        _check_tensor("xw", xw)
        _check_tensor("hOut", hOut)
        _check_tensor("u", u)
        _require(xw.dim() == 3 and hOut.dim() == 3, "xw and hOut must be [Batch, Seq, *]")
        b, s_, g = xw.shape
        h = hOut.shape[2]
        if g != 4 * h:
            raise ShapeError(f"xw must end in 4*hidden = {4 * h} gates (got {g})")
        _require(hOut.shape[0] == b and hOut.shape[1] == s_, "xw and hOut batch/seq differ")
        if list(u.shape) != [h, g]:
            raise ShapeError(f"u must be [{h}, {g}] (got {list(u.shape)})")
        if not (0 <= t < s_):
            raise ShapeError(f"step {t} is outside [0, {s_})")
        _launch("migemm_lstm_recurrent_gates", (xw, hOut, u), _ptr(xw), _ptr(hOut), _ptr(u), b,
                s_, h, int(t))
        return xw

    def LstmHidGates(self, x, w, u, bias, hPrev, hOut, workspace, t):
        """The gate product of step t of lstm_hid_forward (lstm.cl:788-870, gate loop
        :832-844), enqueued by NnClGlob.LstmWithWithState (NnClGlob.cs:1067-1100), in place
        on workspace [S, B, 4H]: workspace[t] = bias + x[:, t] @ w + h_{t-1} @ u, with
        h_{t-1} = hPrev [B, H] at t = 0 and hOut[:, t-1] ([B, S, H]) after. x is [B, S, F],
        w [F, 4H], u [H, 4H], bias [4H]. One launch over the four separate buffers; the
        activations and cell update that follow in the reference kernel are the caller's."""
        for name, v in (("x", x), ("w", w), ("u", u), ("bias", bias), ("hPrev", hPrev),
                        ("hOut", hOut), ("workspace", workspace)):
            _check_tensor(name, v)
        if x.dim() != 3:
            raise ShapeError(f"x must be [Batch, Seq, In] (got {list(x.shape)})")
        b, s_, f = x.shape
        if not (u.dim() == 2 and u.shape[1] == 4 * u.shape[0]):
            raise ShapeError(f"u must be [hidden, 4*hidden] (got {list(u.shape)})")
        h = u.shape[0]
        g = 4 * h
        if list(w.shape) != [f, g]:
            raise ShapeError(f"w must be [{f}, {g}] (got {list(w.shape)})")
        if bias.numel() != g:
            raise ShapeError(f"bias must have {g} elements (got {bias.numel()})")
        if list(hPrev.shape) != [b, h]:
            raise ShapeError(f"hPrev must be [{b}, {h}] (got {list(hPrev.shape)})")
        if list(hOut.shape) != [b, s_, h]:
            raise ShapeError(f"hOut must be [{b}, {s_}, {h}] (got {list(hOut.shape)})")
        if list(workspace.shape) != [s_, b, g]:
            raise ShapeError(f"workspace must be [{s_}, {b}, {g}] (got {list(workspace.shape)})")
        if not (0 <= t < s_):
            raise ShapeError(f"step {t} is outside [0, {s_})")
        _launch("migemm_lstm_hid_gates", (x, w, u, bias, hPrev, hOut, workspace), _ptr(x),
                _ptr(w), _ptr(u), _ptr(bias), _ptr(hPrev), _ptr(hOut), _ptr(workspace), b, s_,
                f, h, int(t))
        return workspace

    def LstmGemmGradX(self, allGradGates, w, xShape):
        """grad_X (shape xShape) = allGradGates[T, 4H] @ w[F, 4H]^T: stage 2 of
        NnClGlob.LstmBackward (NnClGlob.cs:967-994, lstm_gemm_grad_x lstm.cl:372-457)."""
        _check_tensor("allGradGates", allGradGates)
        _check_tensor("w", w)
        if w.dim() != 2:
            raise ShapeError(f"w must be [in_features, 4*hidden] (got {list(w.shape)})")
        f, g = w.shape
        if allGradGates.shape[-1] != g:
            raise ShapeError(f"allGradGates must end in {g} gates (got {list(allGradGates.shape)})")
        t = allGradGates.numel() // g
        gx = torch.empty(list(xShape), dtype=torch.float32, device=w.device)
        if gx.numel() != t * f:
            raise ShapeError(f"xShape {list(xShape)} does not hold [{t}, {f}]")
        _launch("migemm_lstm_gemm_grad_x", (w, allGradGates, gx), _ptr(allGradGates), _ptr(w),
                _ptr(gx), t, f, g)
        return gx

    def LstmGemmGradWeights(self, x, hOut, allGradGates, gradW, gradU, gradBias):
        """Stage 3 of NnClGlob.LstmBackward (NnClGlob.cs:996-1024, lstm_gemm_grad_weights
        lstm.cl:459-636), accumulating in place like w.Grad / u.Grad / bias.Grad there:
        gradW += X^T G, gradU += H_prev^T G (h_{t-1} of the same sequence, 0 at its first
        step), gradBias += sum over tokens of G. x is [B, S, F], hOut [B, S, H]."""
        for name, t in (("x", x), ("hOut", hOut), ("allGradGates", allGradGates),
                        ("gradW", gradW), ("gradU", gradU), ("gradBias", gradBias)):
            _check_tensor(name, t)
        _require(x.dim() == 3 and hOut.dim() == 3, "x and hOut must be [Batch, Seq, *]")
        b, s_, f = x.shape
        h = hOut.shape[2]
        _require(hOut.shape[0] == b and hOut.shape[1] == s_, "x and hOut batch/seq differ")
        _require(allGradGates.numel() == b * s_ * 4 * h, "allGradGates must be [B*S, 4*hidden]")
        if gradW.numel() != f * 4 * h:
            raise ShapeError(f"gradW must hold [{f}, {4 * h}]")
        if gradU.numel() != h * 4 * h:
            raise ShapeError(f"gradU must hold [{h}, {4 * h}]")
        if gradBias.numel() != 4 * h:
            raise ShapeError(f"gradBias must hold {4 * h} values")
        _launch("migemm_lstm_gemm_grad_weights", (x, hOut, allGradGates, gradW, gradU, gradBias),
                _ptr(x), _ptr(hOut), _ptr(allGradGates), _ptr(gradW), _ptr(gradU),
                _ptr(gradBias), b, s_, f, h)
        return gradW, gradU, gradBias

    def Sum(self, x, axis, keepDims=False):
        """Sum over one axis, ascending order (NnClGlob.cs:1595-1664)."""
        _check_tensor("x", x)
        ax = axis + x.dim() if axis < 0 else axis
        if ax < 0 or ax >= x.dim():
            raise IndexError(f"axis {axis} is out of range for a {x.dim()}-D tensor")
        outer = 1
        for s in x.shape[:ax]:
            outer *= s
        inner = 1
        for s in x.shape[ax + 1:]:
            inner *= s
        if keepDims:
            shape = list(x.shape)
            shape[ax] = 1
        elif x.dim() == 1:
            shape = [1]
        else:
            shape = [s for i, s in enumerate(x.shape) if i != ax]
        y = torch.empty(shape, dtype=torch.float32, device=x.device)
        _launch("migemm_reduce_sum_axis", (x, y), _ptr(x), _ptr(y), outer, x.shape[ax], inner)
        return y

    # -------------------------------------------------------------- Python names
    def bmm(self, A, B):
        """Python reference bmm (nncl_glob.py:110-147): equal batches required."""
        _check_tensor("A", A)
        _check_tensor("B", B)
        _require(A.dim() == 3 and B.dim() == 3,
                 "BMM expects 3-D tensors [Batch, M/K, K/N]")
        _require(A.shape[0] == B.shape[0], "the Batch dimension of A and B must match")
        return self.Bmm(A, B)

    def permute(self, x, axes):
        """Python reference permute (nncl_glob.py:148-174); synchronous like it."""
        y = self.Permute(x, axes)
        _synchronize(x)
        return y

    def bmm_backward(self, grad_output, A, B):
        """(grad_A, grad_B) = (dC @ B^T, A^T @ dC) (nncl_glob.py:283-312), computed with
        the NT and TN kernels instead of permute + bmm."""
        grad_A = self.BmmPermute(grad_output, B, transA=False, transB=True)
        grad_B = self.BmmPermute(A, grad_output, transA=True, transB=False)
        _synchronize(A)
        return grad_A, grad_B

    # ------------------------------------------------------------- extra forms
    def linear_weight_grad(self, x, grad_output):
        """dW[1,K,N] = sum_b x_b^T @ dY_b in one TN GEMM over batch*M rows (the
        BmmPermute(transA) + Sum(axis 0) pair of LinearOp.cs:37-38)."""
        _check_tensor("x", x)
        _check_tensor("grad_output", grad_output)
        _require(x.dim() == 3 and grad_output.dim() == 3, "expects 3-D tensors")
        batch, m, k = x.shape
        _require(grad_output.shape[0] == batch and grad_output.shape[1] == m,
                 "x and grad_output must share [Batch, M]")
        n = grad_output.shape[2]
        dw = torch.empty((1, k, n), dtype=torch.float32, device=x.device)
        _launch("migemm_linear_weight_grad", (x, grad_output, dw), _ptr(x), _ptr(grad_output),
                _ptr(dw), m, k, n, batch)
        return dw

    @staticmethod
    def reserve_workspace(stream, nbytes):
        """Sizes the library workspace of `stream` (a torch.cuda.Stream) to at least nbytes
        per buffer before it is captured into a HIP graph: a capture allocates nothing, and a
        split GEMM captured on a stream whose workspace is too small fails with
        MIGEMM_ERR_WORKSPACE (migemm_workspace_reserve)."""
        _native.call("migemm_workspace_reserve", ctypes.c_void_p(stream.cuda_stream),
                     int(nbytes))

    def gemm(self, a, b, transA=False, transB=False, bias=None, out=None):
        """General 2-D / batched entry point: out = op(a) @ op(b) (+ bias)."""
        _check_tensor("a", a)
        _check_tensor("b", b)
        squeeze = a.dim() == 2 and b.dim() == 2
        a3 = a.unsqueeze(0) if a.dim() == 2 else a
        b3 = b.unsqueeze(0) if b.dim() == 2 else b
        _require(a3.dim() == 3 and b3.dim() == 3, "gemm expects 2-D or 3-D tensors")
        batch = max(a3.shape[0], b3.shape[0])
        _require(a3.shape[0] in (batch, 1) and b3.shape[0] in (batch, 1), "batch mismatch")
        m, k = (a3.shape[2], a3.shape[1]) if transA else (a3.shape[1], a3.shape[2])
        kb, n = (b3.shape[2], b3.shape[1]) if transB else (b3.shape[1], b3.shape[2])
        if k != kb:
            raise ShapeError(f"inner dimensions differ: {k} != {kb}")
        if bias is not None:
            _check_tensor("bias", bias)
            if bias.numel() != n:
                raise ShapeError(f"bias must have {n} elements")
        if out is None:
            out = torch.empty((batch, m, n), dtype=torch.float32, device=a.device)
        else:
            _check_tensor("out", out)
            _require(out.numel() == batch * m * n, "out has the wrong size")
        sA = 0 if a3.shape[0] == 1 else a3.shape[1] * a3.shape[2]
        sB = 0 if b3.shape[0] == 1 else b3.shape[1] * b3.shape[2]
        _launch("migemm_gemm_strided_batched", (a, b, out) + ((bias,) if bias is not None else ()),
                int(transA), int(transB), m, n, k, _ptr(a3), a3.shape[2], sA, _ptr(b3),
                b3.shape[2], sB, _ptr(bias) if bias is not None else None, _ptr(out), n, m * n,
                batch)
        return out.view(m, n) if squeeze else out

    # ---------------------------------------------------------------- serving in 8 bits
    # The reference has no counterpart. Activations are float32 or bfloat16; rows of a larger
    # tensor (a slice of a fused projection) are taken as they lie. All of these only enqueue
    # work on the current stream; nothing is read back, and no gradient is recorded.
    def QuantizeRows(self, x):
        """(values, scales) of x[..., K] in 8 bits, a scale for each row: scales [rows] =
        max |x| / 127 over the row, values int8 [rows, K rounded up to 16] = x / scale rounded
        half to even, the added columns 0. A weight [out, in] is laid out by it once; a row
        with a value that is not finite gets the scale NaN."""
        code = _check_rows("x", x)
        k = x.shape[-1] if x.dim() else 0
        if x.dim() < 1 or k < 1:
            raise ShapeError(f"x must have rows of at least one value (got {list(x.shape)})")
        x2 = x if x.dim() == 2 else x.reshape(-1, k)
        rows = x2.shape[0]
        values = torch.empty((rows, (k + 15) // 16 * 16), dtype=torch.int8, device=x.device)
        scales = torch.empty(rows, dtype=torch.float32, device=x.device)
        if rows:
            _launch("migemm_quantize_rows", (x2, values, scales), _ptr(x2), code,
                    _row_stride("x", x2), _ptr(values), values.shape[1], _ptr(scales), rows, k)
        return values, scales

    def NormInt8(self, x, weight=None, residual=None, eps=1e-6):
        """(values, scales, sum) of the rows x[..., K] after a residual's addition: sum =
        x + residual of x's type (x itself where residual is None), and in 8 bits, as
        QuantizeRows lays them out, the rows of sum / sqrt(mean(sum^2) + eps) * weight (float32
        [K]; None: ones). They are the a and aScales of MatmulInt8, and the sum is the residual of
        what follows. residual has the shape of x; eps > 0."""
        code = _check_rows("x", x)
        k = x.shape[-1] if x.dim() else 0
        if k < 1:
            raise ShapeError(f"x must have rows of at least one value (got {list(x.shape)})")
        eps = float(eps)
        _require(0.0 < eps < math.inf, "eps must be finite and greater than 0")
        x2 = x if x.dim() == 2 else x.reshape(-1, k)
        rows = x2.shape[0]
        operands = (x2,)
        if weight is not None:
            _check_typed("weight", weight, torch.float32, (k,))
            operands += (weight,)
        r2 = total = None
        if residual is not None:
            if _check_rows("residual", residual) != code or residual.shape != x.shape:
                raise ShapeError(f"residual must be {x.dtype} {list(x.shape)} (got "
                                 f"{residual.dtype} {list(residual.shape)})")
            r2 = residual if x.dim() == 2 else residual.reshape(-1, k)
            total = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
            operands += (r2, total)
        values = x.new_empty((rows, (k + 15) // 16 * 16), dtype=torch.int8)
        scales = x.new_empty(rows, dtype=torch.float32)
        if rows:
            added = (None, 0)
            if r2 is not None:
                added = (_ptr(r2), k if r2.is_contiguous() else _row_stride("residual", r2))
            _launch("migemm_norm_int8", operands + (values, scales), _ptr(x2),
                    k if x2.is_contiguous() else _row_stride("x", x2), *added, code,
                    _ptr(weight) if weight is not None else None, eps,
                    _ptr(total) if total is not None else None, k, _ptr(values),
                    values.shape[1], _ptr(scales), rows, k)
        return values, scales, x if total is None else total

    def MatmulInt8(self, a, aScales, b, bScales, bias=None, dtype=torch.float32, activation=None,
                   gated=False, residual=None):
        """C[M, N] of dtype from c = (a[M, K] @ b[N, K]^T) * aScales[M] * bScales[N] (+ bias[N]):
        int8 rows as QuantizeRows or NormInt8 gives them (K a multiple of 16, at most 131071; rows
        may lie further apart than K). The integer sum is exact. In the same launch:
        activation ("relu", "silu", "gelu", "gelu_tanh"; None: C = c) gives C = activation(c);
        gated C = activation(gate) * up, with b [2N, K] (bScales and bias [2N]): N rows of the
        gate, then N of up; residual [M, N] of dtype is added to either. All of it is float32,
        rounded to dtype once."""
        if dtype not in _TYPES:
            raise ShapeError(f"dtype must be float32 or bfloat16 (got {dtype})")
        for name, t in (("a", a), ("b", b)):
            _require(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
            if t.dtype != torch.int8 or t.dim() != 2:
                raise ShapeError(f"{name} must be int8 [rows, K] (got {t.dtype} "
                                 f"{list(t.shape)})")
            _require(t.is_cuda, f"{name} must live on the GPU: there is no CPU fallback")
        m, k = a.shape
        wide = b.shape[0]
        if b.shape[1] != k:
            raise ShapeError(f"inner dimensions differ: {k} != {b.shape[1]}")
        _check_typed("aScales", aScales, torch.float32, (m,))
        _check_typed("bScales", bScales, torch.float32, (wide,))
        if bias is not None:
            _check_typed("bias", bias, torch.float32, (wide,))
        n, closing = _closing(wide, activation, gated)
        c = torch.empty((m, n), dtype=dtype, device=a.device)
        if residual is not None:
            _check_residual(residual, c)
        if m and n:
            if not k:
                raise ShapeError("K must be at least 1")
            extra = (bias,) if bias is not None else ()
            product = (_ptr(a), _row_stride("a", a), _ptr(aScales), _ptr(b), _row_stride("b", b),
                       _ptr(bScales), _ptr(bias) if bias is not None else None)
            out = (_ptr(c), _TYPES[dtype], n, m, n, k)
            if closing is None and residual is None:
                _launch("migemm_matmul_int8", (a, b, aScales, bScales, c) + extra, *product, *out)
            else:
                if residual is not None:
                    extra += (residual,)
                _launch("migemm_matmul_int8_ex", (a, b, aScales, bScales, c) + extra, *product,
                        *(closing or (0, 0)), *_residual_at(residual), *out)
        return c

    def LinearInt8(self, x, weight, scales, bias=None, activation=None, gated=False,
                   residual=None):
        """y[..., N] from x[..., K] @ W^T (+ bias[N], float32) with W [N, K] as QuantizeRows left
        it (weight int8 [N, K rounded up to 16], scales [N]); the rows of x are quantised on
        the way. y has the type of x. activation, gated (W [2N, K]) and residual (y's shape and
        type) as MatmulInt8's. One launch where rows * ceil(K / 4096) <= 3; otherwise
        the quantised rows go through the stream's workspace (reserve_workspace before a
        capture). For inference: the result carries no gradient."""
        code = _check_rows("x", x)
        _check_typed("weight", weight, torch.int8, dim=2)
        wide, kp = weight.shape
        k = x.shape[-1] if x.dim() else 0
        if k < 1 or (k + 15) & -16 != kp:
            raise ShapeError(f"x must end in the weight's features (got {list(x.shape)} and "
                             f"rows of {kp} bytes)")
        _check_typed("scales", scales, torch.float32, (wide,))
        if bias is not None:
            _check_typed("bias", bias, torch.float32, (wide,))
        n, closing = _closing(wide, activation, gated)
        x2 = x if x.dim() == 2 else x.reshape(-1, k)
        m = x2.shape[0]
        y = x.new_empty((m, n))
        if residual is not None:
            if x.dim() != 2:
                _check_rows("residual", residual)
                if residual.shape != x.shape[:-1] + (n,):
                    raise ShapeError(f"residual must be {list(x.shape[:-1]) + [n]} (got "
                                     f"{list(residual.shape)})")
                residual = residual.reshape(m, n)
            _check_residual(residual, y)
        if m and n:
            extra = (bias,) if bias is not None else ()
            layer = (_ptr(x2), code, _row_stride("x", x2), _ptr(weight), kp, _ptr(scales),
                     _ptr(bias) if bias is not None else None)
            out = (_ptr(y), n, m, n, k)
            if closing is None and residual is None:
                _launch("migemm_linear_int8", (x2, weight, scales, y) + extra, *layer, *out)
            else:
                if residual is not None:
                    extra += (residual,)
                _launch("migemm_linear_int8_ex", (x2, weight, scales, y) + extra, *layer,
                        *(closing or (0, 0)), *_residual_at(residual), *out)
        return y if x.dim() == 2 else y.reshape(list(x.shape[:-1]) + [n])

    def CacheTables(self, lengths, counts, table, free, freeCount, tokens, pageSize):
        """The pages and slots of a step that adds counts[i] tokens to each request of
        lengths[i] tokens: (slots [tokens], positions [tokens], starts [requests + 1], the new
        lengths [requests], the pages left [1]), all int32; table [requests, pages a request]
        gets the new pages' numbers, taken from the end of free[0 .. freeCount). Requests are
        packed in order; `tokens` is the size of the step's buffers, tokens past the step's
        end get slot and position -1. A request is admitted if its table row and `tokens` hold
        it and it needs no new page or enough are left after the requests before it; else
        its tokens get -1 and its length stays. The lengths and freeCount given are not
        changed: a caller goes on with the ones returned."""
        requests, columns = _check_table(lengths, table)
        _check_typed("counts", counts, torch.int32, (requests,))
        _check_typed("free", free, torch.int32, dim=1)
        _check_typed("freeCount", freeCount, torch.int32, (1,))
        tokens = int(tokens)
        _require(tokens >= 0, "tokens must not be negative")
        # one buffer: five allocations would cost more than the kernel
        out = lengths.new_empty(2 * tokens + 2 * requests + 2)
        at = _ptr(out)
        rest = at + 8 * tokens
        _launch("migemm_cache_tables", (lengths, counts, table, free, freeCount, out),
                _ptr(lengths), _ptr(counts), requests, _ptr(table), columns, int(pageSize),
                _ptr(free), _ptr(freeCount), free.shape[0], at, at + 4 * tokens, rest,
                rest + 4 * requests + 4, rest + 8 * requests + 4, tokens)
        return out.split_with_sizes((tokens, tokens, requests + 1, requests, 1))

    def CacheSlots(self, lengths, counts, table, tokens, pageSize):
        """(slots [tokens], positions [tokens], starts [requests + 1]) of the tokens lengths[i]
        .. lengths[i] + counts[i] of each request in the pages that its table row names: with
        lengths 0 and the lengths as counts, every cached token."""
        requests, columns = _check_table(lengths, table)
        _check_typed("counts", counts, torch.int32, (requests,))
        tokens = int(tokens)
        _require(tokens >= 0, "tokens must not be negative")
        out = lengths.new_empty(2 * tokens + requests + 1)
        at = _ptr(out)
        _launch("migemm_cache_slots", (lengths, counts, table, out), _ptr(lengths),
                _ptr(counts), requests, _ptr(table), columns, int(pageSize), at,
                at + 4 * tokens, at + 8 * tokens, tokens)
        return out.split_with_sizes((tokens, tokens, requests + 1))

    def CacheRelease(self, finished, lengths, table, free, freeCount, pageSize):
        """Gives the pages of every request with finished[i] != 0 back: added at the end of
        free[0 .. freeCount) (free has room for the whole pool), its table row becomes -1 and
        its length 0. In place. Pages are not counted: set the entries of a page that another
        request goes on using to -1 before."""
        requests, columns = _check_table(lengths, table)
        _check_typed("finished", finished, torch.int32, (requests,))
        _check_typed("free", free, torch.int32, dim=1)
        _check_typed("freeCount", freeCount, torch.int32, (1,))
        _launch("migemm_cache_release", (finished, lengths, table, free, freeCount),
                _ptr(finished), _ptr(lengths), requests, _ptr(table), columns,
                int(pageSize), _ptr(free), free.numel(), _ptr(freeCount))

    def CacheAppend(self, k, v, slots, cache):
        """Writes the keys k and values v [tokens, kv heads, head size] of a step into their
        slots of an Int8Cache (slots of CacheTables; -1 skips a token, wherever it stands;
        the other tokens of one page are neighbours). A page and head whose scale is too small for the new tokens gets
        theirs, and what it holds is rounded anew."""
        code = _check_rows("k", k, 3)
        if _check_rows("v", v, 3) != code:
            raise ShapeError(f"k and v must have one type (got {k.dtype} and {v.dtype})")
        tokens = k.shape[0]
        want = (tokens, cache.kvHeads, cache.headDim)
        if k.shape != want or v.shape != want:
            raise ShapeError(f"k and v must be {list(want)} (got {list(k.shape)} and "
                             f"{list(v.shape)})")
        _check_typed("slots", slots, torch.int32, (tokens,))
        held, place = cache.operands()
        if tokens:
            _launch("migemm_cache_append", (k, v, slots) + held, _ptr(k), _ptr(v), code,
                    _row_stride("k", k), _row_stride("v", v), _ptr(slots), tokens, *place)

    def CacheRead(self, cache, slots, dtype=torch.float32):
        """(k, v) [tokens, kv heads, head size] of dtype: what the cache holds at slots (e.g.
        of CacheSlots), 0 where a slot is -1. For products over a cached context through Bmm."""
        if dtype not in _TYPES:
            raise ShapeError(f"dtype must be float32 or bfloat16 (got {dtype})")
        _check_typed("slots", slots, torch.int32, dim=1)
        held, place = cache.operands()
        tokens = slots.numel()
        k = torch.empty((tokens, cache.kvHeads, cache.headDim), dtype=dtype,
                        device=slots.device)
        v = torch.empty_like(k)
        if tokens:
            _launch("migemm_cache_read", (slots, k, v) + held, *place, _ptr(slots), tokens,
                    _ptr(k), _ptr(v), _TYPES[dtype])
        return k, v

    def CacheAttention(self, q, cache, table, starts, positions, scale=None, maxCount=0,
                       maxLength=0):
        """Causal attention of a step's queries q [tokens, heads, head size] over an Int8Cache:
        query t of request i (starts[i] <= t < starts[i + 1]) sees the request's tokens 0 ..
        positions[t] (its own, already appended, among them), head h the kv head
        h // (heads / kv heads). scale: 1 / sqrt(head size) if None. Tokens without a position
        (-1) or request (before starts[0], past the last start) give 0. starts and positions are
        CacheTables' (starts never descend); maxCount (most tokens of
        one request) and maxLength (longest request) shape the launches if the caller knows
        them, the result does not depend on them. Returns [tokens, heads, head size] of q's
        type."""
        code = _check_rows("q", q, 3)
        tokens, heads, dim = q.shape
        if dim != cache.headDim or heads % cache.kvHeads or not heads:
            raise ShapeError(f"q must be [tokens, a multiple of {cache.kvHeads} heads, "
                             f"{cache.headDim}] (got {list(q.shape)})")
        _check_typed("table", table, torch.int32, dim=2)
        requests, columns = table.shape
        _check_typed("starts", starts, torch.int32, (requests + 1,))
        _check_typed("positions", positions, torch.int32, (tokens,))
        held, place = cache.operands()
        o = q.new_empty((tokens, heads, dim))
        if tokens:
            _launch("migemm_cache_attention", (q, table, starts, positions, o) + held, _ptr(q),
                    code, _row_stride("q", q), *place, _ptr(table), columns, _ptr(starts),
                    _ptr(positions), requests, tokens, heads,
                    dim ** -0.5 if scale is None else float(scale), int(maxCount),
                    int(maxLength), _ptr(o))
        return o

    def Sample(self, logits, uniforms, temperature=1.0, topK=0, topP=1.0, minP=0.0):
        """(tokens int32 [rows], probabilities float32 [rows]): a token for each row of logits
        [rows, vocabulary] (float32 or bfloat16, at most 2^20 tokens) from its random number
        uniforms [rows] in [0, 1) (float32). Tokens stand by logit, largest first, equal ones by
        index, and weigh w = exp((logit - largest) / temperature). minP: those with w < minP weigh
        nothing; topK: so do those beyond the first topK (0: no limit); topP: of the others the
        fewest are kept that hold topP of their sum. The token is the first whose weights up to
        its own are more than uniform times the kept ones' sum; its probability is its share of
        that. temperature 0: the largest logit's first token. Every parameter is a number (topP
        above 0), or a tensor [rows] (float32; topK int32) with one for each row, which is not
        refused (a topP of 0 or less keeps one token, a topK of 0 or less all). Rows that allow no
        token (all -inf), that hold a NaN, or whose uniform or parameter in a tensor is NaN or a
        temperature negative or infinite give token -1 and probability 0; a logit of inf counts as
        the largest float32. Few rows (at most vocabulary / 1024, and at most 128) of 40960 tokens
        or more use the stream's workspace (reserve_workspace before a capture)."""
        code = _check_rows("logits", logits, 2)
        rows, vocab = logits.shape
        _check_typed("uniforms", uniforms, torch.float32, (rows,))
        operands = (logits, uniforms)
        params = []
        for name, v, dtype, low, high in (("temperature", temperature, torch.float32, 0, _MOST),
                                          ("topK", topK, torch.int32, 0, 2 ** 31 - 1),
                                          ("topP", topP, torch.float32, 0, 1),
                                          ("minP", minP, torch.float32, 0, 1)):
            if isinstance(v, torch.Tensor):
                _check_typed(name, v, dtype, (rows,))
                operands += (v,)
                params += (_ptr(v), 0)
            else:
                v = operator.index(v) if dtype is torch.int32 else float(v)
                if not low <= v <= high:
                    raise ShapeError(f"{name} must be in {low}..{high} (got {v})")
                params += (None, v)
        if not vocab:
            raise ShapeError("logits must have at least one token")
        tokens = logits.new_empty(rows, dtype=torch.int32)
        probabilities = logits.new_empty(rows, dtype=torch.float32)
        if rows:
            _launch("migemm_sample", operands + (tokens, probabilities), _ptr(logits), code,
                    _row_stride("logits", logits), rows, vocab, _ptr(uniforms), *params,
                    _ptr(tokens), _ptr(probabilities))
        return tokens, probabilities
