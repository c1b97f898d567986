"""Operator-level convenience wrappers: emit the gfx950 kernel for one
operator instance, compile it once, launch it on torch device tensors.
Shapes are static (baked into the kernel), like every kernel the generator
emits."""
import math
import operator
import threading

import torch

from . import runtime as R


def _need_cuda(*ts):
    for t in ts:
        if not (t.is_cuda and t.is_contiguous()):
            raise ValueError("operands must be contiguous device tensors")


# (operator, every property of the operands that the kernel depends on) -> the bound launch of that kernel.  Nothing in a
# key or a value belongs to one tensor: shapes, types, options and whether the operands are aligned.  A call with kernel
# parameters of its own (cfg) goes through get_kernel each time.  The oldest entries of a program with ever new sizes are dropped; their
# kernels stay loaded.
class _Launches(dict):
    MOST = 4096
    _change = threading.Lock()

    def __setitem__(self, key, launch):
        with self._change:
            while len(self) >= self.MOST and key not in self:
                del self[next(iter(self))]
            super().__setitem__(key, launch)


_bound = _Launches()


def _into(run, shape=None, dtype=None):
    """A bound launch whose last pointer is the result: a function of the operand tensors (and numbers) that allocates the result,
    of that shape and type on the first operand's device, or like the first operand, launches and returns it.  The result is a plain
    tensor; where a subclass of the operand decides about it (torch.empty_like), the caller allocates."""
    native = getattr(run, "result", None)
    if native is not None:
        return native(shape, dtype)

    def call(*operands):
        first = operands[0]
        out = torch.empty_like(first) if shape is None else torch.empty(shape, dtype=dtype, device=first.device)
        pointers = [t.data_ptr() for t in operands if isinstance(t, torch.Tensor)]
        run(*pointers, out.data_ptr(), *operands[len(pointers):])
        return out
    return call


# storage type of the row kernels (their arithmetic is fp32 throughout): the kernels' F16 parameter
_STORAGE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def layernorm(x, gamma, beta, axis, eps=1e-5, gelu=False, out=None, **cfg):
    _need_cuda(x, gamma, beta)
    # plain numbers: a key must not hold an object that can change, nor find 1 for a refused 1.0
    axis, eps, gelu = operator.index(axis), float(eps), int(gelu)
    key = ("layernorm", x.shape, x.dtype, gamma.shape, gamma.dtype, beta.shape, beta.dtype, axis, eps, gelu)
    hit = None if cfg else _bound.get(key)
    if hit is None:
        run = _layernorm_kernel(x, gamma, beta, axis, eps, gelu, cfg).bind()
        hit = run, _into(run)
        if not cfg:
            _bound[key] = hit
    if out is None:
        if type(x) is torch.Tensor:
            return hit[1](x, gamma, beta)
        out = torch.empty_like(x)
    hit[0](x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), out.data_ptr())
    return out


def _layernorm_kernel(x, gamma, beta, axis, eps, gelu, cfg):
    axis = axis + x.dim() if axis < 0 else axis
    rows = int(math.prod(x.shape[:axis])) if axis > 0 else 1
    n = x.numel() // rows
    if x.dtype not in _STORAGE or gamma.dtype != x.dtype or beta.dtype != x.dtype:
        raise ValueError("the LayerNorm kernel takes fp32, IEEE half or bfloat16 tensors of one type")
    return R.get_kernel("layernorm", ROWS=rows, N=n, NG=gamma.numel(), NB=beta.numel(), EPS=float(eps),
                        GELU=int(gelu), F16=_STORAGE[x.dtype], **cfg)


_CTYPE = {torch.float32: "float", torch.int32: "int", torch.float16: "_Float16", torch.bfloat16: "__bf16"}


def elementwise(x, op, inplace=False, out_dtype=None, **cfg):
    _need_cuda(x)
    out_dtype, inplace = out_dtype or x.dtype, int(inplace)
    key = ("elementwise", x.numel(), op, inplace, x.dtype, out_dtype)
    hit = None if cfg else _bound.get(key)
    if hit is None:
        run = R.get_kernel("elementwise", N=x.numel(), OP=op, INPLACE=int(inplace), IN_T=_CTYPE[x.dtype],
                           OUT_T=_CTYPE[out_dtype], **cfg).bind()
        hit = run, None if inplace or out_dtype != x.dtype else _into(run)
        if not cfg:
            _bound[key] = hit
    run, into = hit
    if inplace:
        run(x.data_ptr())
        return x if out_dtype == x.dtype else x.view(out_dtype)
    if into is not None and type(x) is torch.Tensor:
        return into(x)
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    run(x.data_ptr(), y.data_ptr())
    return y


def _aligned(a, b):
    """What both operands' addresses are multiples of: 16, 4, or less (1)."""
    low = a.data_ptr() | b.data_ptr()
    return 1 if low & 3 else 4 if low & 15 else 16


def _alignment(aligned):
    """The kernel parameters for it.  Direct loads into LDS take any address that is a multiple of four bytes, so those give
    the kernels that whole tiles get without looking (fp32 1024^3 off a 16-byte boundary: 21 us, 26 through registers; bf16
    4096^3 with row-major weights: 112 and 129); the forms for all sizes split rows into 16-byte chunks and are for ALIGN = 16.
    Other addresses go through registers."""
    return {"ALIGN": 16} if aligned == 16 else {} if aligned == 4 else {"D2L": 0}


_FAMILY = {torch.float32: "gemm_f32", torch.float64: "gemm_f64", torch.bfloat16: "gemm_bf16", torch.float16: "gemm_bf16"}


def batched_matmul(a, b, trans_a=False, trans_b=False, out_dtype=None, **cfg):
    """a: [..., m, k] (or [..., k, m] when trans_a), b: [..., k, n] (or [..., n, k]).  out_dtype None: fp64 for fp64
    operands, fp32 for all others; a type the operands' kernel family does not write raises."""
    _need_cuda(a, b)
    trans_a, trans_b = bool(trans_a), bool(trans_b)
    key = ("matmul", a.shape, b.shape, a.dtype, b.dtype, trans_a, trans_b, out_dtype, _aligned(a, b))
    hit = None if cfg else _bound.get(key)
    if hit is None:
        hit = _matmul_launch(a, b, trans_a, trans_b, out_dtype, cfg)
        if not cfg:
            _bound[key] = hit
    return hit(a, b)


def _matmul_launch(a, b, trans_a, trans_b, out_dtype, cfg):
    """The bound kernel, which allocates its result."""
    if a.dtype != b.dtype or a.dtype not in _FAMILY:
        raise ValueError("unsupported operand dtypes")
    batch = int(math.prod(a.shape[:-2])) if a.dim() > 2 else 1
    m, k = (a.shape[-1], a.shape[-2]) if trans_a else (a.shape[-2], a.shape[-1])
    n, k2 = (b.shape[-2], b.shape[-1]) if trans_b else (b.shape[-1], b.shape[-2])
    if k != k2:
        raise ValueError("incompatible K dimensions")
    extra, align = {}, {}
    if out_dtype is None:
        out_dtype = torch.float64 if a.dtype == torch.float64 else torch.float32
    if a.dtype in (torch.bfloat16, torch.float16):
        if out_dtype not in (torch.float32, a.dtype):
            raise ValueError("a 16-bit GEMM writes fp32 or its operands' type")
        extra["OUT_BF16"] = int(out_dtype == a.dtype)       # a 16-bit result, of the operands' type
        if a.dtype == torch.float16:
            extra["F16"] = 1
        align = _alignment(_aligned(a, b))
    elif a.dtype == torch.float64:
        if out_dtype != torch.float64:
            raise ValueError("fp64 GEMM writes fp64")
    elif out_dtype != torch.float32:
        raise ValueError("fp32 GEMM writes fp32")
    else:
        align = _alignment(_aligned(a, b))
    # (the caller's parameters go before the alignment's, and may not name any other)
    kern = R.get_kernel(_FAMILY[a.dtype], M=m, N=n, K=k, BATCH=batch, TA=int(trans_a), TB=int(trans_b),
                        **extra, **{**align, **cfg})
    run = (lambda *p: kern.launch(*p)) if kern.info["workspace_bytes"] else kern.bind()
    return _into(run, tuple(a.shape[:-2]) + (m, n), out_dtype)


def matmul_fp8(a, b, scale_a, scale_b, trans_a=False, trans_b=True, out_dtype=torch.float32, **cfg):
    """(scale_a * op(a)) (scale_b * op(b)) with fp8 e4m3 operands, one fp32 scale per tensor and fp32
    accumulation.  a: [..., m, k] (or [..., k, m] when trans_a), b: [..., k, n] (or [..., n, k] when
    trans_b, the default: both operands k-contiguous, no transposition on the way into LDS)."""
    _need_cuda(a, b)
    trans_a, trans_b = bool(trans_a), bool(trans_b)
    key = ("matmul_fp8", a.shape, b.shape, a.dtype, b.dtype, trans_a, trans_b, out_dtype, _aligned(a, b))
    hit = None if cfg else _bound.get(key)
    if hit is None:
        hit = _matmul_fp8_launch(a, b, trans_a, trans_b, out_dtype, cfg)
        if not cfg:
            _bound[key] = hit
    return hit(a, b, float(scale_a), float(scale_b))


def _matmul_fp8_launch(a, b, trans_a, trans_b, out_dtype, cfg):
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise ValueError("operands must be float8_e4m3fn")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("output must be fp32 or bf16")
    batch = int(math.prod(a.shape[:-2])) if a.dim() > 2 else 1
    m, k = (a.shape[-1], a.shape[-2]) if trans_a else (a.shape[-2], a.shape[-1])
    n, k2 = (b.shape[-2], b.shape[-1]) if trans_b else (b.shape[-1], b.shape[-2])
    if k != k2:
        raise ValueError("incompatible K dimensions")
    kern = R.get_kernel("gemm_fp8", M=m, N=n, K=k, BATCH=batch, TA=int(trans_a), TB=int(trans_b),
                        OUT_BF16=int(out_dtype == torch.bfloat16), **{**_alignment(_aligned(a, b)), **cfg})
    return _into(kern.bind(scalars=2), tuple(a.shape[:-2]) + (m, n), out_dtype)


def matmul(a, b, **cfg):
    return batched_matmul(a, b, **cfg)


def fmha(q, k, v, scale=None, causal=False, out_dtype=None, **cfg):
    """softmax(scale * q k^T [+ causal mask]) v over [B, H, S, D] operands, all fp32, all bf16 or all IEEE half; the
    result has their type (default) or is fp32.  fp32 operands run both products on the fp32 MFMA (fmha_f32)."""
    _need_cuda(q, k, v)
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("q, k, v must share one [B, H, S, D] shape")
    if not (q.dtype == k.dtype == v.dtype and q.dtype in (torch.float32, torch.bfloat16, torch.float16)):
        raise ValueError("the fused attention kernels take fp32, bf16 or IEEE half operands")
    out_dtype = q.dtype if out_dtype is None else out_dtype
    if out_dtype not in (q.dtype, torch.float32):
        raise ValueError("output must have the operands' type or be fp32")
    scale, causal = (None if scale is None else float(scale)), int(causal)
    key = ("fmha", q.shape, q.dtype, scale, causal, out_dtype)
    run = None if cfg else _bound.get(key)
    if run is None:
        b, h, s, d = q.shape
        scale = d ** -0.5 if scale is None else scale
        if q.dtype == torch.float32:
            kern = R.get_kernel("fmha_f32", B=b, H=h, S=s, D=d, CAUSAL=int(causal), SCALE=scale, **{"FILL": 1, **cfg})
        else:
            kern = R.get_kernel("fmha_bf16", B=b, H=h, S=s, D=d, CAUSAL=int(causal), SCALE=scale,
                                OUT_BF16=int(out_dtype == q.dtype), F16=int(q.dtype == torch.float16), **{"FILL": 1, **cfg})
        run = _into(kern.bind(), tuple(q.shape), out_dtype)
        if not cfg:
            _bound[key] = run
    return run(q, k, v)


def binary(x, y, op, inplace=False, **cfg):
    """x op y (Add, Sub, Mul, Div, Pow; Equal and Greater give a bool tensor) on two fp32 or two IEEE half tensors
    with numpy-style broadcasting."""
    _need_cuda(x, y)
    if x.dtype not in (torch.float32, torch.float16) or y.dtype != x.dtype:
        raise ValueError("the binary kernel takes two fp32 or two IEEE half operands")
    inplace = int(inplace)
    key = ("binary", x.shape, y.shape, x.dtype, op, inplace)
    hit = None if cfg else _bound.get(key)
    if hit is None:
        hit = _binary_launch(x, y, op, inplace, cfg)
        if not cfg:
            _bound[key] = hit
    if inplace:
        hit(x.data_ptr(), y.data_ptr())
        return x
    return hit(x, y)


def _binary_launch(x, y, op, inplace, cfg):
    shape = torch.broadcast_shapes(x.shape, y.shape)

    def strides(t):
        out, run = [0] * len(shape), 1
        for i in range(t.dim()):
            extent = t.shape[t.dim() - 1 - i]
            if extent != 1:
                out[len(shape) - 1 - i] = run
            run *= extent
        return ",".join(map(str, out))

    k = R.get_kernel("binary", OP=op, DIMS=",".join(map(str, shape)), SA=strides(x), SB=strides(y), INPLACE=int(inplace),
                     F16=int(x.dtype == torch.float16), **cfg)
    return k.bind() if inplace else _into(k.bind(), tuple(shape), torch.bool if op in ("Equal", "Greater") else x.dtype)


def gather(x, indices, axis=0, **cfg):
    """out[o.., i.., r..] = x[o.., indices[i..], r..]: dimension `axis` of x is replaced by the dimensions of
    `indices` (int64; a single index, shape (1,), drops the dimension).  Indices outside the axis are clamped.
    `cfg` overrides kernel parameters (BLOCK, UNROLL)."""
    _need_cuda(x, indices)
    if indices.dtype != torch.int64:
        raise ValueError("gather indices must be int64")
    axis = operator.index(axis)
    if not -x.dim() <= axis < x.dim():
        raise ValueError("axis out of range")
    key = ("gather", x.shape, x.dtype, indices.shape, axis)
    hit = None if cfg else _bound.get(key)
    if hit is None:
        hit = _gather_launch(x, indices, axis, cfg)
        if not cfg:
            _bound[key] = hit
    return hit(x, indices)


def _gather_launch(x, indices, axis, cfg):
    axis %= x.dim()
    outer = 1
    for d in x.shape[:axis]:
        outer *= d
    inner = 1
    for d in x.shape[axis + 1:]:
        inner *= d
    single = tuple(indices.shape) == (1,)
    shape = tuple(x.shape[:axis]) + (() if single else tuple(indices.shape)) + tuple(x.shape[axis + 1:])
    kern = R.get_kernel("gather", OUTER=outer, AXIS=x.shape[axis], NIDX=indices.numel(), INNER=inner, ESIZE=x.element_size(), **cfg)
    return _into(kern.bind(), shape, x.dtype)


def softmax(x, inplace=False):
    """softmax over the last axis of an fp32, IEEE half or bfloat16 tensor (fp32 arithmetic)."""
    _need_cuda(x)
    if x.dtype not in _STORAGE:
        raise ValueError("the softmax kernel takes fp32, IEEE half or bfloat16 operands")
    inplace = int(inplace)
    key = ("softmax", x.shape, x.dtype, inplace)
    hit = _bound.get(key)
    if hit is None:
        n = x.shape[-1]
        run = R.get_kernel("softmax", ROWS=x.numel() // n, N=n, INPLACE=int(inplace), F16=_STORAGE[x.dtype]).bind()
        _bound[key] = hit = run, None if inplace else _into(run)
    if inplace:
        hit[0](x.data_ptr())
        return x
    if type(x) is torch.Tensor:
        return hit[1](x)
    y = torch.empty_like(x)
    hit[0](x.data_ptr(), y.data_ptr())
    return y



# ---- a decoding step: pages, the cache in 8 bits, attention over it, weights of 4 bits ----

def _into_last(run, *results):
    """_into for a kernel whose other arguments are pointers and whole numbers in any order: its results, each a (shape, dtype), are the last
    ones; several are given as a tuple."""
    if hasattr(run, "results"):
        return run.result(*results[0]) if len(results) == 1 else run.results(*results)

    def call(*operands):
        device = operands[0].device
        outs = tuple([torch.empty(shape, dtype=dtype, device=device) for shape, dtype in results])
        run(*[t.data_ptr() if isinstance(t, torch.Tensor) else t for t in operands], *[t.data_ptr() for t in outs])
        return outs if len(outs) > 1 else outs[0]
    return call


def _on_device(*ts):
    for t in ts:
        if not t.is_cuda:
            raise ValueError("operands must be device tensors")


def _vectors(dtype, *ts):
    for t in ts:
        if not (t.is_cuda and t.is_contiguous() and t.dtype == dtype):
            raise ValueError("expected contiguous device tensors of type %s" % dtype)


def page_slots(lengths, added, table, free, page_size, tokens):
    """Page tables and slots of one step's tokens, on the device alone.

    lengths, added: int32 [B], the tokens that each request has in the cache and gets now; table: int32 [B, W], the pages of each request,
    continued in place; free: int32 [F], free pages, handed out from the front, earlier requests first.  tokens: rows of the step,
    sum(added) or more (padding).  Returns (slots int64 [tokens], positions int32 [tokens], starts int32 [B + 1], lengths + added int32
    [B], number of pages taken int32 [1]): slot = page * page_size + place in the page, what cache_write takes; -1 for padding and for
    tokens that have no page, because `free` or the table is too short.  starts and the new lengths are what cache_attention takes."""
    page_size, tokens = operator.index(page_size), operator.index(tokens)
    key = ("page_slots", R.signature(lengths, added), R.row_signature(table, free), page_size, tokens)
    run = _bound.get(key)
    if run is None:
        _bound[key] = run = _page_slots_launch(lengths, added, table, free, page_size, tokens)
    return run(lengths, added, table, free, table.shape[0], tokens, table.shape[1], table.stride(0), free.shape[0])


def _page_slots_launch(lengths, added, table, free, page_size, tokens):
    _vectors(torch.int32, lengths, added, free)
    if lengths.dim() != 1 or lengths.shape != added.shape or free.dim() != 1 or table.dim() != 2 or table.shape[0] != lengths.shape[0]:
        raise ValueError("lengths and added are [B], table is [B, W], free is [F]")
    if not table.is_cuda or table.dtype != torch.int32 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError("the table must be an int32 device tensor with rows of neighbouring entries")
    if not 1 <= page_size <= 0x7FFFFFFF or tokens < 0 or tokens > 0x7FFFFFFF:
        raise ValueError("bad page size or number of tokens")
    batch = table.shape[0]
    # two tokens a lane, as far as that needs no more workgroups than the part has CUs
    kern = R.get_kernel("page_slots", PAGE=page_size, BLOCK=1024 if batch > 256 or tokens > 512 else 256)
    i32 = torch.int32
    return _into_last(kern.bind(grid=(max(1, min(256, -(-tokens // 2048))),)), ((tokens,), torch.int64), ((tokens,), i32), ((batch + 1,), i32), ((batch,), i32),
                      ((1,), i32))


def _cache_strides(cache, scale):
    """Strides of page, token and head of a cache [pages, page, heads, d]."""
    if cache.dim() != 4 or cache.dtype != torch.float8_e4m3fn or (cache.stride(3) != 1 and cache.shape[3] > 1):
        raise ValueError("a cache is a float8_e4m3fn device tensor [pages, page, heads, d] with neighbouring d")
    pages, page, heads, d = cache.shape
    if pages < 1 or pages > 0x7FFFFFFF or page < 16 or page > 256 or page & (page - 1) or d % 32 or not 32 <= d <= 256:
        raise ValueError("a cache has pages of 16, 32, 64, 128 or 256 tokens and a head dimension that is a multiple of 32 up to 256")
    strides = cache.stride()[:3]
    if cache.data_ptr() % 16 or any(s % 16 for s in strides):
        raise ValueError("the rows of a cache must start on multiples of 16 bytes")
    if tuple(scale.shape) != (pages, heads):
        raise ValueError("a cache has one scale per page and head, [pages, heads]")
    return strides


def _row_strides(x, cache, types):
    """Strides of token and head of rows [tokens, heads, d]."""
    if x.dim() != 3 or x.dtype not in types or x.stride(2) != 1 or x.shape[2] != cache.shape[3]:
        raise ValueError("rows are [tokens, heads, d] device tensors with neighbouring d, which is the cache's")
    size = x.element_size()
    if x.data_ptr() % 16 or x.stride(0) * size % 16 or x.stride(1) * size % 16:
        raise ValueError("rows must start on multiples of 16 bytes")
    return x.stride(0), x.stride(1)


def cache_write(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    """Writes new keys and values into a paged cache in 8 bits, in place.

    k, v: [tokens, heads, d], fp32, IEEE half or bfloat16; k_cache, v_cache: float8_e4m3fn [pages, page, heads, d] in any order in memory;
    k_scale, v_scale: fp32 [pages, heads]; slots: int64 [tokens], page * page_size + place in the page, a token with another slot (-1) is
    left out.  The tokens of a page stand together and in order, as page_slots gives them.  A page's scale is the least power of two by
    which its rows fit the format; where a page has earlier rows, these are converted when the scale has to grow.  A page whose
    first row is written is taken to be new.  Infinities become the largest numbers that the scale allows: 0 where all else is 0."""
    key = ("cache_write", R.signature(k, v, k_cache, v_cache, k_scale, v_scale, slots))
    run = _bound.get(key)
    if run is None:
        _bound[key] = run = _cache_write_launch(k, v, k_cache, v_cache, k_scale, v_scale, slots)
    tokens = slots.shape[0]
    if tokens:
        run(k, v, k_cache, v_cache, k_scale, v_scale, slots, tokens, k_cache.shape[0])


def _cache_write_launch(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    _on_device(k, v, k_cache, v_cache)
    _vectors(torch.int64, slots)
    _vectors(torch.float32, k_scale, v_scale)
    if k.shape != v.shape or k.dtype != v.dtype or k_cache.shape != v_cache.shape:
        raise ValueError("keys and values, and their caches, must have one shape and type")
    ks, vs = _cache_strides(k_cache, k_scale), _cache_strides(v_cache, v_scale)
    xk, xv = _row_strides(k, k_cache, _STORAGE), _row_strides(v, v_cache, _STORAGE)
    tokens, heads, d = k.shape
    if heads != k_cache.shape[2] or tuple(slots.shape) != (tokens,) or tokens > 0x7FFFFE00:
        raise ValueError("one slot per token, and the cache's heads, are needed")
    # tokens of a wavefront, which takes the pages they lead one after the other: us for tokens of a page each and of whole pages (8 heads of 128)
    # 128 tokens: one 3.5 and 4, four 5.2 and 3.3;  512: one 6.2 and 8.2, four 6.8 and 4.1, sixteen 15 and 3.6;  9000 of whole pages: 58, 29, 12.5
    win = 1 if tokens <= 128 else 4 if tokens <= 2048 else 16
    kern = R.get_kernel("cache_write", H=heads, D=d, PAGE=k_cache.shape[1], F16=_STORAGE[k.dtype], WIN=win, KP=ks[0], KT=ks[1], KH=ks[2],
                        VP=vs[0], VT=vs[1], VH=vs[2], XKT=xk[0], XKH=xk[1], XVT=xv[0], XVH=xv[1])
    run = kern.bind(grid=(max(1, -(-2 * heads * -(-tokens // win) // 4)),))
    return run if hasattr(run, "results") else lambda *a: run(*[x.data_ptr() if isinstance(x, torch.Tensor) else x for x in a])


def cache_read(cache, scale, slots, dtype=torch.bfloat16):
    """Rows of a paged cache in 8 bits: [tokens, heads, d] in fp32, IEEE half or bfloat16 for slots int64 [tokens]; zeros for a slot that is
    none of the cache's (-1)."""
    key = ("cache_read", R.signature(cache, scale, slots), dtype)
    run = _bound.get(key)
    if run is None:
        _bound[key] = run = _cache_read_launch(cache, scale, slots, dtype)
    return run(cache, scale, slots, slots.shape[0], cache.shape[0])


def _cache_read_launch(cache, scale, slots, dtype):
    _on_device(cache)
    _vectors(torch.int64, slots)
    _vectors(torch.float32, scale)
    if dtype not in _STORAGE or slots.dim() != 1:
        raise ValueError("rows are given in fp32, IEEE half or bfloat16, for slots [tokens]")
    s = _cache_strides(cache, scale)
    page, heads, d = cache.shape[1:]
    tokens = slots.shape[0]
    kern = R.get_kernel("cache_read", H=heads, D=d, PAGE=page, F16=_STORAGE[dtype], KP=s[0], KT=s[1], KH=s[2])
    return _into_last(kern.bind(grid=(max(1, -(-tokens * heads * d // 2048)),)), ((tokens, heads, d), dtype))


def cache_attention(q, k_cache, v_cache, k_scale, v_scale, table, lengths, starts=None, scale=None, cap=None, window=None, slopes=None, **cfg):
    """Attention of new tokens over a paged cache in 8 bits, which holds their own keys and values already.

    q: [tokens, heads, d], IEEE half or bfloat16, heads a multiple of the cache's; caches and scales as for cache_write; table: int32
    [B, W], the pages of each request; lengths: int32 [B], its keys.  starts: int32 [B + 1], rising from 0: the rows of request b are
    starts[b] to starts[b + 1], its last tokens; None: one row each.  Returns [tokens, heads, d] in q's type; rows that see no key,
    and rows behind the last request's, are zeros.
      score = scale * q.k (scale: d^-0.5), then cap * tanh(score / cap), then + slopes[head] * (key's position - row's), slopes fp32
      [heads]; a row sees the keys up to its own position, of these the last `window`.
    Entries of the table behind a request's length have no effect; keys on pages that are not the cache's count as not there.  `cfg`
    overrides kernel parameters (RB, SHARE, WAVES, WHOLE, GRID, LEAST, OCC; SPLIT: whether probabilities keep what their
    rounding to 11 bits leaves, by default for half precision)."""
    scale, cap, window = None if scale is None else float(scale), float(cap or 0.0), operator.index(window or 0)
    key = ("cache_attention", R.signature(q, k_cache, v_cache, k_scale, v_scale, table, lengths, starts, slopes), scale, cap, window)
    hit = None if cfg else _bound.get(key)
    if hit is None:
        hit = _cache_attention_launch(q, k_cache, v_cache, k_scale, v_scale, table, lengths, starts, scale, cap, window, slopes, cfg)
        if not cfg:
            _bound[key] = hit
    run, join, floats = hit
    if not q.shape[0]:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    batch, width = table.shape
    part = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else 0
    out = run(q, k_cache, v_cache, k_scale, v_scale, table, lengths, 0 if starts is None else starts, 0 if slopes is None else slopes, part, q.shape[0], batch,
              width, table.stride(0), k_cache.shape[0])
    if join is not None:
        join(part.data_ptr(), out.data_ptr())
    return out


def _cache_attention_launch(q, k_cache, v_cache, k_scale, v_scale, table, lengths, starts, scale, cap, window, slopes, cfg):
    _on_device(q, k_cache, v_cache, table)
    _vectors(torch.float32, k_scale, v_scale, *(() if slopes is None else (slopes,)))
    _vectors(torch.int32, lengths, *(() if starts is None else (starts,)))
    ks, vs = _cache_strides(k_cache, k_scale), _cache_strides(v_cache, v_scale)
    if k_cache.shape != v_cache.shape:
        raise ValueError("the caches of keys and values must have one shape")
    if max(ks[1], vs[1]) >= 1 << 27:
        raise ValueError("neighbouring tokens of a page must lie less than 2^27 bytes apart")
    qs = _row_strides(q, k_cache, (torch.float16, torch.bfloat16))
    tokens, heads, d = q.shape
    page, kv_heads = k_cache.shape[1:3]
    if heads % kv_heads:
        raise ValueError("the heads of q must be a multiple of the cache's")
    if table.dim() != 2 or table.dtype != torch.int32 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError("the table must be an int32 device tensor [B, W] with rows of neighbouring entries")
    batch, width = table.shape
    # (positions have 32 bits in the kernel, which looks up the pages of up to 96 steps ahead)
    if batch < 1 or width < 1 or width * page > 0x7FFF0000 or tokens > 0x7FFF0000 or tuple(lengths.shape) != (batch,):
        raise ValueError("lengths is [B] and table [B, W], neither B nor W being 0")
    if starts is None and tokens != batch:
        raise ValueError("without starts there is one row per request")
    if starts is not None and tuple(starts.shape) != (batch + 1,):
        raise ValueError("starts is [B + 1]")
    if slopes is not None and tuple(slopes.shape) != (heads,):
        raise ValueError("slopes is [heads]")
    group = heads // kv_heads
    if not 0.0 <= cap < math.inf or window < 0:
        raise ValueError("cap and window must not be negative")
    if cap > 2.0 ** 40:                 # (scores up to 2^27 are what they are to fp32)
        cap = 0.0
    if window >= width * page:          # (none is left out; and a row's position less the window has 32 bits)
        window = 0
    params = dict(H=kv_heads, D=d, PAGE=page, G=group, F16=int(q.dtype == torch.float16), STARTS=int(starts is not None), CAP=cap, WINDOW=window,
                  SLOPES=int(slopes is not None), SCALE=d ** -0.5 if scale is None else scale, KP=ks[0], KT=ks[1], KH=ks[2], VP=vs[0], VT=vs[1], VH=vs[2],
                  QT=qs[0], QH=qs[1], **_cache_attention_form(batch, tokens, kv_heads, group, d, width * page, q.dtype == torch.float16))
    if not cfg.keys() <= {"RB", "WAVES", "SHARE", "GRID", "LEAST", "OCC", "WHOLE", "SPLIT"}:
        raise ValueError("unknown kernel parameters")
    params.update(cfg)
    blocks = params["RB"] * (params["WAVES"] if params["SHARE"] else 1)
    tiles = kv_heads * -(-group // (16 * blocks))         # of a token's heads
    # the kernel counts the units of keys of all tiles in 32 bits
    of, unit = 16 * blocks // min(group, 16 * blocks), 64 if params["SHARE"] else 32 * params["WAVES"]
    if (tokens // of + batch + 1) * ((width * page + of) // unit + 1) > 0x7FFF0000:
        raise ValueError("too many rows times keys for one launch")
    kern = R.get_kernel("cache_attention", **params)
    if params["WHOLE"]:
        # with starts, every request's first tile and what the tokens fill behind it, however they are spread (also behind the last request)
        whole = batch if starts is None else max(1, min(batch + 1, tokens) + tokens // (16 * blocks // min(group, 16 * blocks)))
        return _into_last(kern.bind(grid=(whole * tiles,)), (tuple(q.shape), q.dtype)), None, 0
    shares = kern.info["grid"][0]
    # for each share four whole numbers, and two parts of a tile: its sums, and maximum and sum of the probabilities of each row
    floats = shares * (4 + 2 * (16 * blocks * d + 32 * blocks))
    join = None if shares == tiles else R.get_kernel("cache_join", **params).bind()
    return _into_last(kern.bind(), (tuple(q.shape), q.dtype)), join, floats


def _cache_attention_form(batch, tokens, kv_heads, group, d, keys, half):
    """The tiles and who takes what of them; `keys`: what a request's row of the table has room for.

    A tile has 16 rows of a kv head, whose keys are split between the wavefronts of a workgroup.  Where the average request has more than 32
    rows, or more than 16 of 256 numbers, which registers hold no more keys beside, it has 64 or 128 rows, 16 or 32 (RB) to a wavefront,
    and the wavefronts share the keys (SHARE).  About GRID workgroups take equal shares
    of all keys, so that a few long requests fill the part and a tile may lie in several shares, whose results a second launch joins;
    where requests are short, a workgroup takes one tile (WHOLE), with as many wavefronts as its keys and the number of tiles ask for.
    Measured, in us (8 kv heads of 128, 4 heads to each, bf16; lengths spread up to `keys`, a third of it on average):
      512 tiles, 512 keys: a tile each 10.2, shares 15.5;  4096 tiles: 52, 70;  512 tiles, 1024 keys: 14.2, 21.1;  4096: 94, 101;
      1024 tiles, 2048 keys: 55.3, 54.2;  4096 keys: 102, 90
      a tile each, 4096 tiles, of 16 keys: one wavefront 11.5, two 16.1, four 25.1;  512 keys: 55, 52, 56;  64 tiles, 512 keys: 14.7, 9.1, 6.8
      8 prompts of up to 300 behind up to 600 keys: shared keys with 16 rows a wavefront 41, 32 rows 49, keys split 58;  2 of 1000 behind 6000:
      202, 167, 195;  64 of up to 16 tokens behind 1000: 35, 54, 44
      32 heads to one kv head: 8 of up to 32000 keys: keys split, 16 rows a tile 21.6, 32 rows 26.9, shared 26.2;  16 of 16000 of 256: 38, 61, 32
      2 of 500 behind 4000, 8 heads of 256 to a kv head: half precision 16 rows a wavefront 140, 32 rows 212;  bfloat16, 32 rows: 138"""
    rows = group * max(1, -(-tokens // batch))
    share = int(rows > (32 if d <= 128 else 16))
    blocks = 2 if share and rows * keys >= 1 << 21 and not (half and d > 128) else 1
    tiles = batch * kv_heads * -(-group // 16)
    whole = int(not share and (keys <= 512 or (keys <= 1024 and tiles >= 512)))
    waves = 4
    if whole and keys <= 512:
        waves = (1 if keys <= 64 else 2) if tiles > 512 else 2 if keys <= 64 else 4
    return dict(RB=blocks, SHARE=share, WHOLE=whole, WAVES=waves, GRID=256 if blocks == 2 and d > 128 else 512)


def matmul_q4(x, w, scale, zero=None, out_dtype=None, **cfg):
    """x times the transpose of a matrix of 4-bit numbers: y[..., n] = sum over k of x[..., k] * scale[n, k / group] * (code[n, k] - zero).

    x: [..., K], IEEE half or bfloat16; w: uint8 [N, K / 2], the code of an even k in the low four bits; scale: [N, K / group], fp32 or x's
    type, group 32, 64 or a multiple of 128; zero: uint8 [N, K / group], None for 8.  Codes and x enter the sums unrounded, the sums are fp32; the
    result has x's type (default) or is fp32.  For the few rows of a decoding step: the weights are read once for each 64 rows."""
    key = ("matmul_q4", R.signature(x, w, scale, zero), out_dtype)
    hit = None if cfg else _bound.get(key)
    if hit is None:
        hit = _matmul_q4_launch(x, w, scale, zero, out_dtype, cfg)
        if not cfg:
            _bound[key] = hit
    run, join, rows = hit
    if rows == 0:
        return torch.empty(x.shape[:-1] + (w.shape[0],), dtype=out_dtype or x.dtype, device=x.device)
    out = run(x, w, scale, 0 if zero is None else zero, rows)
    return out if join is None else join(out, rows)


def _matmul_q4_launch(x, w, scale, zero, out_dtype, cfg):
    _need_cuda(x, w, scale, *(() if zero is None else (zero,)))
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if x.dtype not in (torch.float16, torch.bfloat16) or out_dtype not in (x.dtype, torch.float32) or scale.dtype not in (x.dtype, torch.float32):
        raise ValueError("x is IEEE half or bfloat16, result and scales have x's type or are fp32")
    if w.dtype != torch.uint8 or (zero is not None and zero.dtype != torch.uint8):
        raise ValueError("codes and zeros are uint8")
    if x.dim() < 1 or w.dim() != 2 or scale.dim() != 2 or w.shape[1] * 2 != x.shape[-1] or scale.shape[0] != w.shape[0]:
        raise ValueError("x is [..., K], w [N, K / 2], scale [N, K / group]")
    n, k = w.shape[0], x.shape[-1]
    if scale.shape[1] < 1 or k % scale.shape[1] or (zero is not None and zero.shape != scale.shape):
        raise ValueError("scale (and zero) are [N, K / group]")
    group = k // scale.shape[1]
    if group != 32 and group != 64 and group % 128:
        raise ValueError("a group has 32, 64 or a multiple of 128 codes")
    if (x.data_ptr() | w.data_ptr()) % 16:
        raise ValueError("x and w must start on multiples of 16 bytes")
    rows = math.prod(x.shape[:-1])
    if rows > 0x7FFFFF00:
        raise ValueError("too many rows for one launch")
    if rows == 0:
        return None, None, 0
    if not cfg.keys() <= {"MB", "MR", "NT", "WN", "WK", "SPLIT"}:
        raise ValueError("unknown kernel parameters")
    params = dict(N=n, K=k, GROUP=group, F16=int(x.dtype == torch.float16), ZERO=int(zero is not None), SCALE_F32=int(scale.dtype == torch.float32),
                  OUT_F32=int(out_dtype == torch.float32), **{**_matmul_q4_form(rows, n, k, group), **cfg})
    kern = R.get_kernel("gemm_q4", **params)
    shape, split = tuple(x.shape[:-1]) + (n,), kern.info["grid"][2]
    grid = (kern.info["grid"][0], -(-rows // (16 * params["MB"])), split)
    if split == 1:
        return _into_last(kern.bind(grid=grid), (shape, out_dtype)), None, rows
    join = R.get_kernel("gemm_q4_join", **params).bind(grid=(-(-rows * n // 256),))
    return _into_last(kern.bind(grid=grid), ((split, rows, n), torch.float32)), _into_last(join, (shape, out_dtype)), rows


def _matmul_q4_form(rows, n, k, group):
    """The tiles and the splitting of k, by the columns of a workgroup and the rows of X that every workgroup reads again.

    Up to 16 rows, a wavefront's 16 columns are a workgroup while few workgroups read few rows (a product with its neighbours' would need
    fewer, but wait for one another), else 32 or 48, where those are no more workgroups than units, or 64; more rows take 64 columns and two shares of k in a workgroup, or, where there is more
    to do, 128 columns, or 256, 32 to a wavefront, where 128 are more workgroups than units.  A form whose workgroups do not fill the 256
    units splits k, at two launches' price, where a wavefront has four steps of 256 k or more.  Measured, in us (bf16, groups of 128):
      rows 1, N = K = 4096: 16 columns 4.2, 64 columns with k split 6.2;  1, N 32000, K 4096: 17.5, 17.3
      rows 16, N = K = 4096: 6.0, 7.1;  4, N 11008, K 4096: 7.9, 8.2;  8: 9.5, 8.9, 48 columns 8.2;  16, half with zeros: 64 columns 10.9, 48 9.9
      rows 16, N 8192, K 4096: 64 columns 9.1, 32 columns 7.4;  N 14336: 64 columns 10.5, 48 columns 15.5
      rows 32, N = K = 4096: 64 columns 8.2, 256 columns 9.0;  64: 11.9, 12.6;  128: 15.9, 15.7
      rows 32, N 4096, K 11008: 64 columns 15.2, 128 columns 14.0;  64: 24, 20.1;  128: 37, 28.0
      rows 64, N 32000, K 4096: 64 columns 52, 128 columns 37.2, 256 columns 38.6;  128: 89, 61.8, 49.9
      rows 64, N 1024, K 4096: k in four 9.9, in eight 8.2;  N = K = 1024: in one 7.5, in two 7.3"""
    blocks = min(4, -(-rows // 16))
    form = dict(MB=blocks, NT=1, WN=4, WK=2)
    if blocks == 1:
        form["MR"] = 1 << (rows - 1).bit_length()
        tall = -(-n // 16)
        if tall <= 768 or tall <= 1024 and tall * form["MR"] <= 4096:
            form.update(NT=1 if tall * form["MR"] <= 4096 else -(-tall // 256), WN=1, WK=8)
        else:
            form.update(NT=2, WN=2, WK=4)
    elif n * k * -(-rows // 64) >= 1 << 25 or (blocks == 4 and group < 128):        # (64 rows, two shares and their small groups' scales: LDS is too small)
        form.update(NT=1 if -(-n // 128) * -(-rows // 64) <= 256 else 2, WN=8, WK=1)
    workgroups = -(-n // (16 * form["NT"] * form["WN"])) * -(-rows // (16 * blocks))
    steps = -(-k // 256) // form["WK"]
    form["SPLIT"] = max(1, min(256 // workgroups, steps, 64)) if form["WN"] > 1 and steps >= 4 else 1
    return form
