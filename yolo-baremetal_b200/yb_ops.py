"""The text-decoder operators of include/yb_lm.h on torch CUDA tensors.

    attend = Attention(heads, kv_heads, head_dim, torch.bfloat16, causal=True, cap=50.0)
    qk_norm_rope(q, k, q_weight, k_weight, inv_freq, q_out=q, k_out=k_cache, v=v, v_out=v_cache, start=start)
    o = attend(q, k_cache, v_cache, k_len=k_len)
    token, logprob = sample(logits, u, temperature=t, top_k=k, top_p=p)

Every call runs on the current torch stream of its tensors' device and does
not synchronize; outputs that are not given are allocated.  Tensors of another
device, type or shape than an operator takes raise ValueError, as do tensors
that require gradients outside torch.no_grad() (the operators have none); what
the library refuses raises YBError.  The semantics stand in yb_lm.h.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

import yolo_b200 as yb

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# The argument structures of yb_lm.h, field for field.
_ATTN = struct.Struct("@9P12q8i2f")
_QK = struct.Struct("@12P18q9i2f0q")
_SAMPLE = struct.Struct("@8Pq3i0q")


def _fail(msg: str):
    raise ValueError(msg)


def _need(t, name: str, index: int, dtype, shape) -> int:
    """Data pointer of a contiguous tensor of this CUDA device, type and shape; 0 for None."""
    if t is None:
        return 0
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    _fail(f"{name}: contiguous {dtype} of shape {tuple(shape)} on cuda:{index} expected, "
          f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _heads(t, name: str, index: int, dtype, shape) -> tuple:
    """Strides (batch, row, head) of a [B, rows, heads, D] tensor whose last dimension is contiguous."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index:
        _fail(f"{name}: {dtype} of shape {tuple(shape)} on cuda:{index} expected, "
              f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    s = t.stride()
    if s[3] != 1 and shape[3] > 1:
        _fail(f"{name}: the last dimension must be contiguous")
    return s[:3]


def _writable(t, name: str) -> None:
    """Refuses an output whose elements share memory with one another."""
    if not t.is_contiguous() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        _fail(f"{name}: an output must not be expanded")


def _no_gradients(name: str, *tensors) -> None:
    """Refuses tensors through which autograd would expect a gradient: the results would silently have none."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _fail(f"{name}: no gradients; call it under torch.no_grad(), or with detached tensors")


def _cuda(t, name: str) -> int:
    if not t.is_cuda:
        _fail(f"{name}: a CUDA tensor expected, got {t.device}")
    return t.get_device()


def _public_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# The handle of the current stream without a Python stream object around it.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _call(f, args, index: int) -> int:
    """Calls an entry point that runs on the current device, on the tensors' device and stream."""
    if torch.cuda.current_device() == index:
        return f(args, _stream(index))
    with torch.cuda.device(index):
        return f(args, _stream(index))


class Attention:
    """yb_attn_*: attention with optional score cap, distance bias, document and prefix masks.

    One object serves any batch and length, on any stream; its handle lives on `device` (default: the current one).
    Make it before a stream capture, and keep it while a graph that holds its calls is replayed."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, dtype, scale: float | None = None, cap: float = 0.0,
                 causal: bool = False, device=None):
        if dtype not in (torch.float16, torch.bfloat16):
            _fail(f"attention: float16 or bfloat16, got {dtype}")
        if heads < 1 or kv_heads < 1 or heads % kv_heads or head_dim < 8 or head_dim > 128 or head_dim % 8:
            _fail("attention: heads a multiple of kv_heads, head_dim a multiple of 8 in [8, 128]")
        self.heads, self.kv_heads, self.head_dim, self.dtype = int(heads), int(kv_heads), int(head_dim), dtype
        self.scale = float(head_dim) ** -0.5 if scale is None else float(scale)
        self.cap, self.causal = float(cap), bool(causal)
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        else:
            device = torch.device(device)
            if device.type != "cuda":
                _fail(f"attention: a CUDA device expected, got {device}")
            if device.index is None:
                device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self._scratch = {}  # bytes by (B, Sq, Sk)
        self._h = C.c_void_p()
        yb.check(yb.lib().yb_attn_create(self.device.index, C.byref(self._h)), "yb_attn_create")

    def close(self) -> None:
        if self._h:
            h, self._h = self._h, C.c_void_p()
            yb.check(yb.lib().yb_attn_destroy(h), "yb_attn_destroy")

    def __del__(self):
        try:
            # close() synchronizes, which would end a stream capture under way with an error; the few bytes stay.
            if not torch.cuda.is_current_stream_capturing():
                self.close()
        except Exception:
            pass

    def check(self) -> None:
        """Synchronizes and raises if a kernel gave up a bounded wait; rows of the calls since the last check may then
        be wrong."""
        yb.check(yb.lib().yb_attn_check(self._h), "yb_attn_check")

    def __call__(self, q, k, v, out=None, q_len=None, k_len=None, prefix=None, key_range=None, slopes=None):
        """q [B, Sq, heads, D], k and v [B, Sk, kv_heads, D] -> out [B, Sq, heads, D].

        q_len, k_len, prefix int32 [B]; key_range int32 [B, Sq, 2]; slopes float32 [heads].  Rows past q_len keep
        what `out` holds (zeros where it is allocated here).  Does not synchronize: only check() tells of a kernel that
        gave up a wait."""
        index, dt = self.device.index, self.dtype
        if q.dim() != 4 or k.dim() != 4:
            _fail("attention: q, k and v have four dimensions")
        _no_gradients("attention", q, k, v, slopes, out)
        B, Sq, _, _ = q.shape
        Sk = k.shape[1]
        qs = _heads(q, "q", index, dt, (B, Sq, self.heads, self.head_dim))
        ks = _heads(k, "k", index, dt, (B, Sk, self.kv_heads, self.head_dim))
        vs = _heads(v, "v", index, dt, k.shape)
        if out is None:
            make = torch.empty if q_len is None else torch.zeros
            out = make((B, Sq, self.heads, self.head_dim), dtype=dt, device=self.device)
        os = _heads(out, "out", index, dt, q.shape)
        _writable(out, "out")
        i32 = torch.int32
        args = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                          _need(q_len, "q_len", index, i32, (B,)), _need(k_len, "k_len", index, i32, (B,)),
                          _need(prefix, "prefix", index, i32, (B,)),
                          _need(key_range, "key_range", index, i32, (B, Sq, 2)),
                          _need(slopes, "slopes", index, torch.float32, (self.heads,)), *qs, *ks, *vs, *os,
                          _DTYPE[dt], B, Sq, Sk, self.heads, self.kv_heads, self.head_dim, self.causal, self.scale,
                          self.cap)
        n = self._scratch.get((B, Sq, Sk))
        if n is None:
            size = C.c_size_t()
            yb.check(yb.lib().yb_attn_workspace(self._h, args, C.byref(size)), "yb_attn_workspace")
            n = size.value
            if len(self._scratch) < 4096:
                self._scratch[(B, Sq, Sk)] = n
        # Scratch from torch's allocator: its own for each call in flight and for each captured graph.
        ws = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
        st = yb.lib().yb_attn_run(self._h, args, ws.data_ptr() if n else None, n, _stream(index))
        if st:
            yb.check(st, "yb_attn_run")
        return out


def qk_norm_rope(q, k, q_weight, k_weight, inv_freq, q_out=None, k_out=None, v=None, v_out=None, start=None,
                 length=None, positions=None, eps: float = 1e-6, weight_add: float = 0.0, interleaved: bool = False):
    """yb_qk_norm_rope: q [B, S, Hq, D], k (and v) [B, S, Hkv, D] normed per head and rotated.

    k_out (and v_out) [B, rows, Hkv, D] may be caches, written from row start[b] on.  Weights float32 [D] or None,
    inv_freq float64 [R/2] (R rotated dimensions), start and length int32 [B], positions int32 [B, S].
    Returns (q_out, k_out)."""
    dev, dt, where = _cuda(q, "q"), q.dtype, q.device
    if dt not in _DTYPE:
        _fail(f"qk_norm_rope: float32, float16 or bfloat16, got {dt}")
    if q.dim() != 4 or k.dim() != 4:
        _fail("qk_norm_rope: q and k have four dimensions")
    _no_gradients("qk_norm_rope", q, k, v, q_weight, k_weight, inv_freq, q_out, k_out, v_out)
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    qs = _heads(q, "q", dev, dt, (B, S, Hq, D))
    ks = _heads(k, "k", dev, dt, (B, S, Hkv, D))
    if (v is None) != (v_out is None):
        _fail("qk_norm_rope: v and v_out go together")
    make = torch.empty if length is None else torch.zeros
    if q_out is None:
        q_out = make((B, S, Hq, D), dtype=dt, device=where)
    if k_out is None:
        if start is not None:
            _fail("qk_norm_rope: start needs k_out")
        k_out = make((B, S, Hkv, D), dtype=dt, device=where)
    if k_out.dim() != 4:
        _fail("qk_norm_rope: k_out has four dimensions")
    rows = k_out.shape[1]
    qos = _heads(q_out, "q_out", dev, dt, q.shape)
    kos = _heads(k_out, "k_out", dev, dt, (B, rows, Hkv, D))
    _writable(q_out, "q_out")
    _writable(k_out, "k_out")
    vs = vos = (0, 0, 0)
    if v is not None:
        vs = _heads(v, "v", dev, dt, k.shape)
        vos = _heads(v_out, "v_out", dev, dt, k_out.shape)
        _writable(v_out, "v_out")
    if inv_freq.dim() != 1:
        _fail("qk_norm_rope: inv_freq has one dimension")
    half = inv_freq.shape[0]
    i32, f32 = torch.int32, torch.float32
    args = _QK.pack(q.data_ptr(), k.data_ptr(), 0 if v is None else v.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                    0 if v is None else v_out.data_ptr(), _need(q_weight, "q_weight", dev, f32, (D,)),
                    _need(k_weight, "k_weight", dev, f32, (D,)),
                    _need(inv_freq, "inv_freq", dev, torch.float64, (half,)), _need(start, "start", dev, i32, (B,)),
                    _need(length, "length", dev, i32, (B,)), _need(positions, "positions", dev, i32, (B, S)),
                    *qs, *ks, *vs, *qos, *kos, *vos, _DTYPE[dt], B, S, rows, Hq, Hkv, D, 2 * half, bool(interleaved),
                    eps, weight_add)
    st = _call(yb.lib().yb_qk_norm_rope, args, dev)
    if st:
        yb.check(st, "yb_qk_norm_rope")
    return q_out, k_out


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, token=None, logprob=None):
    """yb_sample: one token for each row of logits [B, V] at the random numbers u [B] in [0, 1).

    temperature, top_p, min_p float32 [B], top_k int32 [B].  Returns (token int32 [B], logprob float32 [B])."""
    dev, dt, where = _cuda(logits, "logits"), logits.dtype, logits.device
    if dt not in _DTYPE:
        _fail(f"sample: float32, float16 or bfloat16, got {dt}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        _fail("sample: logits have two dimensions, the last one contiguous")
    _no_gradients("sample", logits, u, temperature, top_p, min_p, logprob)
    B, V = logits.shape
    i32, f32 = torch.int32, torch.float32
    if u is None:
        _fail("sample: u is needed")
    if token is None:
        token = torch.empty(B, dtype=i32, device=where)
    if logprob is None:
        logprob = torch.empty(B, dtype=f32, device=where)
    args = _SAMPLE.pack(logits.data_ptr(), _need(u, "u", dev, f32, (B,)),
                        _need(temperature, "temperature", dev, f32, (B,)), _need(top_k, "top_k", dev, i32, (B,)),
                        _need(top_p, "top_p", dev, f32, (B,)), _need(min_p, "min_p", dev, f32, (B,)),
                        _need(token, "token", dev, i32, (B,)), _need(logprob, "logprob", dev, f32, (B,)),
                        logits.stride(0), _DTYPE[dt], B, V)
    st = _call(yb.lib().yb_sample, args, dev)
    if st:
        yb.check(st, "yb_sample")
    return token, logprob
