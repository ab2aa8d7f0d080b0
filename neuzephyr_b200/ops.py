"""Torch-tensor conveniences over the C ABI (device memory and the current stream come
from torch; every computation is a libnzb kernel). Used by the tests and the benchmark."""
import collections
import ctypes

import torch

from . import _capi as C

_ws_cache = {}


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _workspace(nbytes, device):
    """Grow-only scratch buffer per device (stream-ordered reuse on torch's current stream)."""
    buf = _ws_cache.get(device)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)
        _ws_cache[device] = buf
    return buf


def _check_f32_cuda(*ts):
    for t in ts:
        if t is None:
            continue
        if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
            raise ValueError("expected contiguous float32 CUDA tensors")


def gemm_workspace_bytes(desc):
    n = ctypes.c_size_t(0)
    C.check(C.lib().nzb_gemm_workspace_bytes(ctypes.byref(desc), ctypes.byref(n)))
    return n.value


def gemm(A, B, out=None, transA=False, transB=False, bias=None, bias_mode=C.BIAS_NONE, relu=False,
         accumulate=False):
    """C = op(A) @ op(B) for 2-D row-major float32 tensors through nzb_gemm."""
    _check_f32_cuda(A, B, bias, out)
    M, K = (A.shape[1], A.shape[0]) if transA else A.shape
    K2, N = (B.shape[1], B.shape[0]) if transB else B.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=A.device)
    d = C.GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.lda, d.ldb, d.ldc = A.shape[1], B.shape[1], N
    d.transA, d.transB = int(transA), int(transB)
    d.batch[0] = d.batch[1] = 1
    d.accumulate, d.relu = int(accumulate), int(relu)
    d.bias_mode = bias_mode if bias is not None else C.BIAS_NONE
    d.bias_ld = N
    ws = _workspace(gemm_workspace_bytes(d), A.device)
    C.check(C.lib().nzb_gemm(ctypes.byref(d), _ptr(A), _ptr(B), _ptr(out), _ptr(bias), _ptr(ws), ws.numel(),
                             _stream()))
    return out


def gemm_host(hA, hB, hC=None, transB=False, bias=None, bias_mode=C.BIAS_NONE, relu=False, device=None):
    """C = A @ op(B) with A, B, C (and bias) in host memory (pinned for overlap) through nzb_gemm_host:
    copies in, staging + GEMM per row block, and copies out are pipelined on three streams. The call
    is asynchronous on torch's current stream; synchronise it before reading hC."""
    for t in (hA, hB, hC, bias):
        if t is not None and (t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError("expected contiguous float32 host tensors")
    device = device or torch.device("cuda", torch.cuda.current_device())
    M, K = hA.shape
    K2, N = (hB.shape[1], hB.shape[0]) if transB else hB.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    if hC is None:
        hC = torch.empty((M, N), dtype=torch.float32).pin_memory()
    d = C.GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.lda, d.ldb, d.ldc = hA.shape[1], hB.shape[1], N
    d.transA, d.transB = 0, int(transB)
    d.batch[0] = d.batch[1] = 1
    d.relu = int(relu)
    d.bias_mode = bias_mode if bias is not None else C.BIAS_NONE
    d.bias_ld = N
    n = ctypes.c_size_t(0)
    C.check(C.lib().nzb_gemm_host_workspace_bytes(ctypes.byref(d), ctypes.byref(n)))
    ws = _workspace(n.value, device)
    C.check(C.lib().nzb_gemm_host(ctypes.byref(d), _ptr(hA), _ptr(hB), _ptr(hC), _ptr(bias), _ptr(ws), ws.numel(),
                                  _stream()))
    return hC


def gemm_f16(A16, B16, M, N, K, out=None, bias=None, bias_mode=C.BIAS_NONE, relu=False, accumulate=False):
    """GEMM on pre-staged K-major fp16 operands A16 [M][ldk], B16 [N][ldk] (nzb_gemm_f16)."""
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=A16.device)
    d = C.GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.ldc = N
    d.batch[0] = d.batch[1] = 1
    d.accumulate, d.relu = int(accumulate), int(relu)
    d.bias_mode = bias_mode if bias is not None else C.BIAS_NONE
    d.bias_ld = N
    C.check(C.lib().nzb_gemm_f16(ctypes.byref(d), _ptr(A16), _ptr(B16), A16.shape[1], _ptr(out), _ptr(bias),
                                 _stream()))
    return out


def _ws4(A, B, Cs):
    n = ctypes.c_size_t(0)
    C.check(C.lib().nzb_tensorcore_gemm_workspace_bytes(C.shape4(A.shape), C.shape4(B.shape), C.shape4(Cs),
                                                        ctypes.byref(n)))
    return n.value


def tensorcore_gemm(A, B, out=None):
    """4-D batched forward GEMM with N/C broadcast (the iTensorCoreGEMM seam)."""
    _check_f32_cuda(A, B, out)
    sc = (max(A.shape[0], B.shape[0]), max(A.shape[1], B.shape[1]), A.shape[2], B.shape[3])
    if out is None:
        out = torch.empty(sc, dtype=torch.float32, device=A.device)
    ws = _workspace(_ws4(A, B, out.shape), A.device)
    C.check(C.lib().nzb_tensorcore_gemm(_ptr(A), _ptr(B), _ptr(out), C.shape4(A.shape), C.shape4(B.shape),
                                        C.shape4(out.shape), _ptr(ws), ws.numel(), _stream()))
    return out


def matmul_f32(A, B, out=None):
    """4-D batched product with N/C broadcast at fp32 accuracy (the Tensor::operator* seam, nzb_matmul_f32)."""
    _check_f32_cuda(A, B, out)
    sc = (max(A.shape[0], B.shape[0]), max(A.shape[1], B.shape[1]), A.shape[2], B.shape[3])
    if out is None:
        out = torch.empty(sc, dtype=torch.float32, device=A.device)
    n = ctypes.c_size_t(0)
    C.check(C.lib().nzb_matmul_f32_workspace_bytes(C.shape4(A.shape), C.shape4(B.shape), C.shape4(out.shape),
                                                   ctypes.byref(n)))
    ws = _workspace(n.value, A.device)
    C.check(C.lib().nzb_matmul_f32(_ptr(A), _ptr(B), _ptr(out), C.shape4(A.shape), C.shape4(B.shape),
                                   C.shape4(out.shape), _ptr(ws), ws.numel(), _stream()))
    return out


def gemm_backward(A, B, out):
    """out += A @ B reduced over broadcast batch dims of out (the iGEMMBackward seam)."""
    _check_f32_cuda(A, B, out)
    ws = _workspace(_ws4(A, B, out.shape), A.device)
    C.check(C.lib().nzb_gemm_backward(_ptr(A), _ptr(B), _ptr(out), C.shape4(A.shape), C.shape4(B.shape),
                                      C.shape4(out.shape), _ptr(ws), ws.numel(), _stream()))
    return out


def cast_f32_f16(x, transpose=False):
    """Returns the [rows][ld_out] fp16 operand copy of a 2-D float32 tensor."""
    _check_f32_cuda(x)
    rows, cols = (x.shape[1], x.shape[0]) if transpose else x.shape
    ld_out = (cols + 63) // 64 * 64
    out = torch.empty((rows, ld_out), dtype=torch.float16, device=x.device)
    C.check(C.lib().nzb_cast_f32_f16(_ptr(x), _ptr(out), rows, cols, x.shape[1], ld_out, int(transpose), _stream()))
    return out


def device_status():
    return C.device_status()


def _conv_desc(x_shape, w_shape, Kh, Kw, stride, pad, bias_mode=C.BIAS_NONE, relu=False, accumulate=False):
    d = C.ConvDesc()
    d.N, d.C, d.H, d.W = [int(v) for v in x_shape]
    d.Cout, d.Kh, d.Kw, d.stride, d.pad = int(w_shape[3]), Kh, Kw, stride, pad
    d.weights_per_sample = int(w_shape[0] > 1)
    d.bias_mode, d.relu, d.accumulate = bias_mode, int(relu), int(accumulate)
    return d


def _conv_ws(d, device):
    n = ctypes.c_size_t(0)
    C.check(C.lib().nzb_conv2d_workspace_bytes(ctypes.byref(d), ctypes.byref(n)))
    return _workspace(n.value, device)


def conv2d_forward(x, w, bias, Kh, Kw, stride, pad, relu=False, bias_mode=None, out=None, accumulate=False):
    """y = conv(x, w) (+ bias) (ReLU); x {N,C,H,W}, w {wN,1,C*Kh*Kw,Cout}, bias {1,1,Ho*Wo,Cout} or [Cout].
    accumulate=True adds the result (before ReLU) to the values already in `out`."""
    _check_f32_cuda(x, w, bias, out)
    if bias_mode is None:
        bias_mode = C.BIAS_NONE if bias is None else (C.BIAS_ROW if bias.dim() == 1 else C.BIAS_MATRIX)
    d = _conv_desc(x.shape, w.shape, Kh, Kw, stride, pad, bias_mode, relu, accumulate)
    Ho, Wo = (d.H + 2 * pad - Kh) // stride + 1, (d.W + 2 * pad - Kw) // stride + 1
    if out is None:
        out = torch.empty((d.N, d.Cout, Ho, Wo), dtype=torch.float32, device=x.device)
    ws = _conv_ws(d, x.device)
    C.check(C.lib().nzb_conv2d_forward(ctypes.byref(d), _ptr(x), _ptr(w), _ptr(bias), _ptr(out), _ptr(ws),
                                       ws.numel(), _stream()))
    return out


def conv2d_backward_data(dy, w, x_shape, Kh, Kw, stride, pad, dx):
    """dx += d(conv)/dx (stride 1)."""
    _check_f32_cuda(dy, w, dx)
    d = _conv_desc(x_shape, w.shape, Kh, Kw, stride, pad)
    ws = _conv_ws(d, dy.device)
    C.check(C.lib().nzb_conv2d_backward_data(ctypes.byref(d), _ptr(dy), _ptr(w), _ptr(dx), _ptr(ws), ws.numel(),
                                             _stream()))
    return dx


def conv2d_backward_weight(x, dy, w_shape, Kh, Kw, stride, pad, dw):
    """dw += d(conv)/dw, summed over the batch for shared weights."""
    _check_f32_cuda(x, dy, dw)
    d = _conv_desc(x.shape, w_shape, Kh, Kw, stride, pad)
    ws = _conv_ws(d, x.device)
    C.check(C.lib().nzb_conv2d_backward_weight(ctypes.byref(d), _ptr(x), _ptr(dy), _ptr(dw), _ptr(ws), ws.numel(),
                                               _stream()))
    return dw


def conv2d_backward_bias(dy, x_shape, w_shape, Kh, Kw, stride, pad, dbias):
    _check_f32_cuda(dy, dbias)
    d = _conv_desc(x_shape, w_shape, Kh, Kw, stride, pad)
    C.check(C.lib().nzb_conv2d_backward_bias(ctypes.byref(d), _ptr(dy), _ptr(dbias), _stream()))
    return dbias


def conv2d_backward(x, w, dy, Kh, Kw, stride, pad, dx=None, dw=None, dbias=None, y=None, overwrite_dx=False):
    """The whole backward of one layer through nzb_conv2d_backward (dY read once): accumulates into the
    given dx / dw / dbias ({1,1,Ho*Wo,Cout}); y, when given, is the forward output whose sign masks dY
    (a layer with a fused ReLU). Raises for shapes the one-pass form does not take."""
    _check_f32_cuda(x, w, dy, dx, dw, dbias, y)
    d = _conv_desc(x.shape, w.shape, Kh, Kw, stride, pad)
    d.bias_mode = C.BIAS_MATRIX if dbias is not None else C.BIAS_NONE
    d.relu = int(y is not None)
    d.overwrite_dx = int(overwrite_dx)
    n = ctypes.c_size_t(0)
    C.check(C.lib().nzb_conv2d_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(n)))
    ws = _workspace(n.value, x.device)
    C.check(C.lib().nzb_conv2d_backward(ctypes.byref(d), _ptr(x), _ptr(w), _ptr(y), _ptr(dy), _ptr(dx), _ptr(dw),
                                        _ptr(dbias), _ptr(ws), ws.numel(), _stream()))


def _linear_desc(batch, fin, fout, relu):
    d = C.LinearDesc()
    d.batch, d.in_features, d.out_features, d.relu = batch, fin, fout, int(relu)
    return d


def _linear_ws(d, device):
    n = ctypes.c_size_t(0)
    C.check(C.lib().nzb_linear_workspace_bytes(ctypes.byref(d), ctypes.byref(n)))
    return _workspace(n.value, device)


def linear_forward(x, w, bias=None, relu=False, out=None):
    """y[b][o] = relu(sum_i w[o][i] x[b][i] + bias[o]); x {B,in}, w {out,in}."""
    _check_f32_cuda(x, w, bias, out)
    d = _linear_desc(x.shape[0], x.shape[1], w.shape[0], relu)
    if out is None:
        out = torch.empty((x.shape[0], w.shape[0]), dtype=torch.float32, device=x.device)
    ws = _linear_ws(d, x.device)
    C.check(C.lib().nzb_linear_forward(ctypes.byref(d), _ptr(x), _ptr(w), _ptr(bias), _ptr(out), _ptr(ws),
                                       ws.numel(), _stream()))
    return out


def linear_backward(x, w, y, dy, dx=None, dw=None, dbias=None, relu=False, overwrite_dx=False):
    """dx += dy' w (dx = ... with overwrite_dx), dw += dy'^T x, dbias += colsum(dy'), dy' = dy * (y > 0) if relu."""
    _check_f32_cuda(x, w, y, dy, dx, dw, dbias)
    d = _linear_desc(x.shape[0], x.shape[1], w.shape[0], relu)
    d.overwrite_dx = int(overwrite_dx)
    ws = _linear_ws(d, x.device)
    C.check(C.lib().nzb_linear_backward(ctypes.byref(d), _ptr(x), _ptr(w), _ptr(y), _ptr(dy), _ptr(dx), _ptr(dw),
                                        _ptr(dbias), _ptr(ws), ws.numel(), _stream()))


# ---- token models ------------------------------------------------------------------------------------------
# These work on the device their tensors live on, whichever is current, and take their scratch from torch's
# allocator call by call: calls on several streams, or captured into several graphs, share no buffer. Small calls
# are bound by the host (a launch is 5 us of it), so the checks go by plain integers.

TokenLogprobs = collections.namedtuple("TokenLogprobs", "logprob entropy lse top_logprob top_index")

_F32 = torch.float32
_DTYPES = {torch.float32: C.F32, torch.float16: C.F16, torch.bfloat16: C.BF16}
_INDEX_TYPES = {torch.int32: C.I32, torch.int64: C.I64}


def _launch(device, fn, *args):
    """Calls an entry point on the current stream of device number `device`; the stream is the call's last argument."""
    if device == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc != C.OK:
        C.check(rc)


def _scratch(fn, d, like):
    n = ctypes.c_size_t(0)
    C.check(fn(ctypes.byref(d), ctypes.byref(n)))
    return torch.empty(n.value, dtype=torch.uint8, device=like.device)


def _dtype(t, what):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError("%s: expected float32, float16 or bfloat16, got %s" % (what, t.dtype))
    return code


def _index_type(t, what):
    code = _INDEX_TYPES.get(t.dtype)
    if code is None:
        raise ValueError("%s: expected int32 or int64, got %s" % (what, t.dtype))
    return code


def _row_stride(t, what):
    """Stride between the rows of a matrix whose rows are contiguous."""
    if t.dim() != 2:
        raise ValueError("%s: expected two dimensions, got %d" % (what, t.dim()))
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError("%s: the elements of a row have to be contiguous" % what)
    if rows > 1:
        if ld < cols:
            raise ValueError("%s: rows overlap" % what)
        return ld
    return cols or 1


def _same_device(first, *ts):
    """Number of the CUDA device that all tensors (or None) live on."""
    device = first.get_device()
    if device < 0:
        raise ValueError("expected CUDA tensors")
    for t in ts:
        if t is not None and t.get_device() != device:
            raise ValueError("tensors are on different devices")
    return device


def _vector(t, n, what, dtype=_F32):
    """Checks an optional contiguous vector of n elements; returns its address (None when absent)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError("%s: expected a contiguous %s tensor of %d elements" % (what, dtype, n))
    return t.data_ptr()


def embedding(table, index, scale=1.0, out=None, out_dtype=None):
    """scale * table[index]: rows of table {vocab, dim} by token number (int32 or int64, any shape); the result has
    the shape of index with dim appended. out_dtype: the table's type, or a 16-bit type for a float32 table. An index
    outside the table gives a row of zeros."""
    device = _same_device(table, index, out)
    ld_table = _row_stride(table, "table")
    if not index.is_contiguous():
        index = index.contiguous()
    vocab, dim = table.shape
    shape = index.shape + (dim,)
    if out is None:
        out = table.new_empty(shape) if out_dtype is None else table.new_empty(shape, dtype=out_dtype)
        ld_out = dim
    else:
        if out.shape != shape:
            raise ValueError("out: expected the shape %s" % (tuple(shape),))
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError("out is not of out_dtype")
        if out.dim() == 2:
            ld_out = _row_stride(out, "out")
        elif out.is_contiguous():
            ld_out = dim
        else:
            raise ValueError("out: expected contiguous rows")
    d = C.EmbeddingDesc(index.numel(), vocab, dim, ld_table, ld_out, -1, scale, _dtype(out, "out"), _dtype(table, "table"),
                        _index_type(index, "index"))
    _launch(device, C.lib().nzb_embedding_forward, ctypes.addressof(d), table.data_ptr(), index.data_ptr(), out.data_ptr())
    return out


def embedding_backward(dy, index, dtable, scale=1.0, padding_index=None, overwrite=False):
    """dtable[v] += scale * the sum of the rows of dy whose index is v, in the order of the rows; overwrite=True
    writes dtable instead, with zeros for tokens that do not occur. dtable is float32 {vocab, dim}; tokens equal to
    padding_index, or outside the table, contribute nothing."""
    device = _same_device(dtable, dy, index)
    if dtable.dtype is not _F32:
        raise ValueError("dtable: expected float32")
    ld_table = _row_stride(dtable, "dtable")
    n, (vocab, dim) = index.numel(), dtable.shape
    if dy.shape != index.shape + (dim,):
        raise ValueError("dy: expected the shape %s" % (tuple(index.shape) + (dim,),))
    if not index.is_contiguous():
        index = index.contiguous()
    if dy.dim() != 2:
        dy = dy.reshape(n, dim)
    d = C.EmbeddingDesc(n, vocab, dim, ld_table, _row_stride(dy, "dy"), -1 if padding_index is None else padding_index, scale,
                        _dtype(dy, "dy"), C.F32, _index_type(index, "index"), overwrite)
    L = C.lib()
    ws = _scratch(L.nzb_embedding_backward_workspace_bytes, d, dtable)
    _launch(device, L.nzb_embedding_backward, ctypes.addressof(d), dy.data_ptr(), index.data_ptr(), dtable.data_ptr(),
            ws.data_ptr(), ws.numel())
    return dtable


def layernorm_forward(x, gamma=None, beta=None, eps=1e-5, out=None):
    """Layer norm over the last dimension of x {rows, dim}; gamma and beta are float32 {dim}. Returns y, mean and rstd
    (float32 {rows}, what the backward pass reads). out may be x."""
    device = _same_device(x, gamma, beta, out)
    ld_x = _row_stride(x, "x")
    rows, dim = x.shape
    if out is None:
        out, ld_y = x.new_empty((rows, dim)), dim or 1
    else:
        ld_y = _row_stride(out, "out")
        if out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError("out: expected the shape and type of x")
    mean = x.new_empty(rows, dtype=_F32)
    rstd = torch.empty_like(mean)
    d = C.LayernormDesc(rows, dim, ld_x, ld_y, 0, eps, _dtype(x, "x"))
    _launch(device, C.lib().nzb_layernorm_forward, ctypes.addressof(d), x.data_ptr(), _vector(gamma, dim, "gamma"),
            _vector(beta, dim, "beta"), out.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    return out, mean, rstd


def layernorm_backward(dy, x, mean, rstd, gamma=None, dx=None, dgamma=None, dbeta=None, overwrite_dx=False,
                       overwrite_dparams=False):
    """Adds the gradients of layernorm_forward to the given dx (type of x) and dgamma / dbeta (float32); the overwrite
    flags write instead. mean and rstd are what the forward pass returned. dx may be dy when it is overwritten."""
    device = _same_device(x, dy, mean, rstd, gamma, dx, dgamma, dbeta)
    ld_x, ld_dy = _row_stride(x, "x"), _row_stride(dy, "dy")
    rows, dim = x.shape
    for t, what in ((dy, "dy"), (dx, "dx")):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError("%s: expected the shape and type of x" % what)
    d = C.LayernormDesc(rows, dim, ld_x, ld_dy, 0 if dx is None else _row_stride(dx, "dx"), 0.0, _dtype(x, "x"), overwrite_dx,
                        overwrite_dparams)
    L = C.lib()
    ws = None if dgamma is None and dbeta is None else _scratch(L.nzb_layernorm_backward_workspace_bytes, d, x)
    _launch(device, L.nzb_layernorm_backward, ctypes.addressof(d), dy.data_ptr(), x.data_ptr(), _vector(mean, rows, "mean"),
            _vector(rstd, rows, "rstd"), _vector(gamma, dim, "gamma"), None if dx is None else dx.data_ptr(),
            _vector(dgamma, dim, "dgamma"), _vector(dbeta, dim, "dbeta"), None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel())


def token_logprobs(logits, targets, scale=1.0, top_k=0):
    """Log probabilities of the targets under softmax(scale * logits) for logits {rows, vocab}, with each row's entropy,
    its log-sum-exp (what the backward pass reads) and the top_k likeliest tokens with their log probabilities (equal
    ones by the lower token; top_k <= 32). A target outside [0, vocab) has log probability 0."""
    device = _same_device(logits, targets)
    ld = _row_stride(logits, "logits")
    rows, vocab = logits.shape
    target_ptr = _vector(targets, rows, "targets", targets.dtype)
    logprob = logits.new_empty(rows, dtype=_F32)
    entropy, lse = torch.empty_like(logprob), torch.empty_like(logprob)
    top_logprob, top_index = logprob.new_empty((rows, top_k)), targets.new_empty((rows, top_k))
    d = C.TokenLogprobDesc(rows, vocab, ld, 0, scale, _dtype(logits, "logits"), _index_type(targets, "targets"), top_k)
    _launch(device, C.lib().nzb_token_logprob_forward, ctypes.addressof(d), logits.data_ptr(), target_ptr, logprob.data_ptr(),
            entropy.data_ptr(), lse.data_ptr(), top_logprob.data_ptr() if top_k else None, top_index.data_ptr() if top_k else None)
    return TokenLogprobs(logprob, entropy, lse, top_logprob, top_index)


def token_logprobs_backward(logits, targets, lse, entropy=None, dlogprob=None, dentropy=None, scale=1.0, out=None):
    """Gradient of token_logprobs with respect to the logits, for upstream gradients dlogprob and dentropy (float32
    {rows}, either may be absent); lse and entropy are the forward pass's. out may be logits."""
    device = _same_device(logits, targets, lse, entropy, dlogprob, dentropy, out)
    ld = _row_stride(logits, "logits")
    rows, vocab = logits.shape
    if out is None:
        out, ld_out = logits.new_empty((rows, vocab)), vocab or 1
    else:
        ld_out = _row_stride(out, "out")
        if out.shape != logits.shape or out.dtype != logits.dtype:
            raise ValueError("out: expected the shape and type of logits")
    d = C.TokenLogprobDesc(rows, vocab, ld, ld_out, scale, _dtype(logits, "logits"), _index_type(targets, "targets"))
    _launch(device, C.lib().nzb_token_logprob_backward, ctypes.addressof(d), logits.data_ptr(),
            _vector(targets, rows, "targets", targets.dtype), _vector(lse, rows, "lse"), _vector(entropy, rows, "entropy"),
            _vector(dlogprob, rows, "dlogprob"), _vector(dentropy, rows, "dentropy"), out.data_ptr())
    return out


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def _batch_strides(t, what):
    if t.dim() == 2:
        return _row_stride(t, what), 0
    if t.dim() != 3:
        raise ValueError("%s: expected a matrix or a batch of matrices" % what)
    if 0 in t.shape:
        return t.shape[2] or 1, 0
    ld = _row_stride(t[0], what)
    if t.shape[0] > 1 and t.stride(0) < (t.shape[1] - 1) * ld + t.shape[2]:
        raise ValueError("%s: matrices overlap" % what)
    return ld, t.stride(0)


def orthogonalize(g, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, out=None, out_dtype=None):
    """The matrix (or batch of matrices) g with its singular values brought near 1 by Newton-Schulz products, as the
    Muon optimizer applies them to an update; out_dtype: g's when not given. Before the rounding to out_dtype it is 1e-5 to 6e-5 off
    the 64-bit result (Frobenius norm), up to 1e-3 for matrices of rank one, as a chain of fp32 products is."""
    device = _same_device(g, out)
    ld_g, stride_g = _batch_strides(g, "g")
    if out is None:
        out = g.new_empty(g.shape, dtype=out_dtype)
    elif out.shape != g.shape or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError("out: expected the shape of g and out_dtype")
    ld_out, stride_out = _batch_strides(out, "out")
    batch = g.shape[0] if g.dim() == 3 else 1
    d = C.OrthogonalizeDesc(batch, g.shape[-2], g.shape[-1], ld_g, stride_g, ld_out, stride_out,
                            (ctypes.c_float * 3)(*coefficients), eps, steps, _dtype(g, "g"), _dtype(out, "out"))
    L = C.lib()
    ws = _scratch(L.nzb_orthogonalize_workspace_bytes, d, g)
    _launch(device, L.nzb_orthogonalize, ctypes.addressof(d), g.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel())
    return out


def muon_step(w, momentum, grad, lr, scale=None, mu=0.95, weight_decay=0.0, nesterov=True, steps=5,
              coefficients=NEWTON_SCHULZ, eps=1e-7):
    """One Muon step on contiguous float32 w, momentum and grad ({rows, cols}, or a batch of such):
    momentum = mu * momentum + grad, w = (1 - lr * weight_decay) * w - lr * scale * orthogonalize(u) with u the momentum
    or, with nesterov, grad + mu * momentum. scale: sqrt(max(1, rows / cols)) when not given."""
    device = _same_device(w, momentum, grad)
    _check_f32_cuda(w, momentum, grad)
    if momentum.shape != w.shape or grad.shape != w.shape or w.dim() not in (2, 3):
        raise ValueError("expected three matrices, or batches of matrices, of one shape")
    rows, cols = w.shape[-2:]
    if scale is None:
        scale = max(1.0, rows / max(cols, 1)) ** 0.5
    d = C.OrthogonalizeDesc(w.shape[0] if w.dim() == 3 else 1, rows, cols, cols, rows * cols, cols, rows * cols,
                            (ctypes.c_float * 3)(*coefficients), eps, steps)
    L = C.lib()
    ws = _scratch(L.nzb_muon_workspace_bytes, d, w)
    _launch(device, L.nzb_muon, ctypes.addressof(d), w.data_ptr(), momentum.data_ptr(), grad.data_ptr(), lr, scale, mu,
            weight_decay, int(nesterov), ws.data_ptr(), ws.numel())
    return w
