"""go-whistle's int8 KV numerics (internal/needle/int8.go) and its packed
Linear (internal/needle/linear.go) over libcqhip.

QuantizeRows / Int8Rows.Append (int8.go:116-141) on host arrays or device
tensors, AttendInt8Spans (int8.go:208-272) on device tensors for one or
many independent streams, fakeQuant (int8.go:57-75), and Linear with
WithInt8Input, Apply and ApplyShared on device tensors. Caches of any
type and length (PagedKV), cross-attention to float memories
(cross_attend_dev), the query and key heads' norms with their rotation
(qk_norm_rope_dev), log probabilities (logprobs_dev) and the verification of
drafted tokens (verify_drafts_dev) on device tensors.
"""

import ctypes
import struct
from ctypes import POINTER, c_float, c_int8, c_void_p

import numpy as np

from ._lib import CQPanic, KvPaged, check, lib


def QuantizeRows(x, cols, width):
    """Codes and scales of x, rows of cols values, per chunk of width (host)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if width <= 0 or cols % width != 0:
        raise CQPanic(f"needle: int8 rows of {cols} in chunks of {width}")
    if x.size % cols != 0:
        raise CQPanic(f"needle: {x.size} values are not rows of {cols}")
    rows = x.size // cols
    q = np.zeros(x.size, dtype=np.int8)
    s = np.zeros(rows * (cols // width), dtype=np.float32)
    check(lib().kv_quantize_rows(q.ctypes.data_as(POINTER(c_int8)), s.ctypes.data_as(POINTER(c_float)),
                                 x.ctypes.data_as(POINTER(c_float)), rows, cols, width))
    return q, s


def QuantizeRow(x):
    """QuantizeRow (int8.go:36-55): codes and the scale of one chunk."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    q, s = QuantizeRows(x, x.size, x.size) if x.size else (np.zeros(0, np.int8), np.ones(1, np.float32))
    return q, float(s[0])


def _stream():
    import torch

    return c_void_p(torch.cuda.current_stream().cuda_stream)


def quantize_rows_dev(q, s, x, rows, cols, width):
    """Device form: q int8 [rows*cols], s float32 [rows*cols/width], x float32."""
    check(lib().kv_quantize_rows_dev(c_void_p(q.data_ptr()), c_void_p(s.data_ptr()), c_void_p(x.data_ptr()),
                                     rows, cols, width, _stream()))


def attend_int8_dev(out, q, t, heads, kq, ks, k_cols, qk, vq, vs, v_cols, vd, spans, nk_max, scale, quant_q,
                    batch=1, out_stride=0, q_stride=0, kv_stride=0, s_stride=0, rope=None):
    """AttendInt8Spans on device tensors for `batch` streams (see cqhip.h).
    rope = (cos, sin, qpos): the query heads are first rotated by RoPE at
    row qpos[b*t + i] of the tables."""
    args = [c_void_p(out.data_ptr()), out_stride, c_void_p(q.data_ptr()), q_stride, t, heads,
            c_void_p(kq.data_ptr()), c_void_p(ks.data_ptr()), k_cols, qk, c_void_p(vq.data_ptr()),
            c_void_p(vs.data_ptr()), v_cols, vd, kv_stride, s_stride, c_void_p(spans.data_ptr()), nk_max, float(scale),
            1 if quant_q else 0, batch]
    if rope is None:
        check(lib().kv_attend_int8_dev(*args, _stream()))
    else:
        cos, sin, qpos = rope
        check(lib().kv_attend_int8_rope_dev(*args, c_void_p(cos.data_ptr()), c_void_p(sin.data_ptr()),
                                            c_void_p(qpos.data_ptr()), _stream()))


def append_dev(q, s, x, batch, cols, width, q_stride, s_stride, pos, cap, rope=None):
    """Int8Rows.Append of one row per stream at pos[b] (see cqhip.h); rope =
    (cos, sin): each chunk is first rotated by RoPE at row pos[b]."""
    args = [c_void_p(q.data_ptr()), c_void_p(s.data_ptr()), c_void_p(x.data_ptr()), batch, cols, width, q_stride,
            s_stride, c_void_p(pos.data_ptr()), cap]
    if rope is None:
        check(lib().kv_append_dev(*args, _stream()))
    else:
        cos, sin = rope
        check(lib().kv_append_rope_dev(*args, c_void_p(cos.data_ptr()), c_void_p(sin.data_ptr()), _stream()))


def fake_quant_dev(dst, x, rows, cols, width):
    """fakeQuant (int8.go:57-75) on device tensors: rows of cols values, each
    chunk of width through QuantizeRow and back; dst may be x."""
    check(lib().nd_fake_quant_dev(c_void_p(dst.data_ptr()), c_void_p(x.data_ptr()), rows, cols, width, _stream()))


def sigmoid_gate_dev(out, gate, n):
    """Attention.output's gate (attention.go:245-249) on device tensors:
    gate = sigmoid(gate), out *= gate over n values."""
    check(lib().nd_sigmoid_gate_dev(c_void_p(out.data_ptr()), c_void_p(gate.data_ptr()), n, _stream()))


def rms_unit_dev(dst, x, rows, dim):
    """RMSUnit (norm.go:68-81) on device rows."""
    check(lib().nd_rms_unit_dev(c_void_p(dst.data_ptr()), c_void_p(x.data_ptr()), rows, dim, _stream()))


def mhc_heads_dev(h_pre, h_post, h_res, u, pre_logits, post_logits, res_logits, stream, rows, lanes, dim,
                  affine=None):
    """MHC.forward's heads and block input from the φ logits (mhc.go:204-263)."""
    p = lambda t: c_void_p(t.data_ptr()) if t is not None else None
    check(lib().nd_mhc_heads_dev(p(h_pre), p(h_post), p(h_res), p(u), p(pre_logits), p(post_logits), p(res_logits),
                                 p(stream), rows, lanes, dim, p(affine), _stream()))


def mhc_heads_stacked_dev(h_pre, h_post, h_res, u, logits, stream, rows, lanes, dim, affine=None):
    """mhc_heads_dev with the logits of each row side by side, rows x (2 lanes
    + lanes^2): pre, post, res (one product of the stacked φ matrices)."""
    p = lambda t: c_void_p(t.data_ptr()) if t is not None else None
    check(lib().nd_mhc_heads_stacked_dev(p(h_pre), p(h_post), p(h_res), p(u), p(logits), p(stream), rows, lanes, dim,
                                         p(affine), _stream()))


def mhc_mix_dev(out, stream, h_res, h_post, block_out, u, rows, lanes, dim):
    """MHC.forward's output stream (mhc.go:229-299)."""
    p = lambda t: c_void_p(t.data_ptr())
    check(lib().nd_mhc_mix_dev(p(out), p(stream), p(h_res), p(h_post), p(block_out), p(u), rows, lanes, dim,
                               _stream()))


class HadamardMLP:
    """HadamardMLP (internal/needle/hadamard.go:12-24, 172-310), Whistle's
    Monarch FFN, with its weights on the device: w holds d1, d2, b2, d3, d4,
    w1a..w3b (square factors), cond_v (dim x rank), cond_u (rank x n) and the
    permutations p1, p2 (hada_p1/p2). forward_dev(out, x, rows) runs
    nd_hadamard_mlp_dev on device tensors of rows x dim."""

    def __init__(self, w, device="cuda"):
        import torch

        f32 = lambda a: torch.as_tensor(np.ascontiguousarray(a, np.float32), device=device)
        self.na, self.nb = int(np.shape(w["w1a"])[0]), int(np.shape(w["w1b"])[0])
        self.dim, self.rank = int(np.shape(w["cond_v"])[0]), int(np.shape(w["cond_v"])[1])
        self._vecs = [f32(w[k]) for k in ("d1", "d2", "b2", "d3", "d4")]
        self._facs = [f32(w[f"w{s}{h}"]) for s in (1, 2, 3) for h in ("a", "b")]
        self._cv, self._cu = f32(w["cond_v"]), f32(w["cond_u"])
        self._p = [torch.as_tensor(np.ascontiguousarray(w[k], np.int32), device=device) for k in ("p1", "p2")]
        n = self.na * self.nb
        for k in ("p1", "p2"):
            if sorted(np.asarray(w[k]).tolist()) != list(range(n)):
                raise CQPanic(f"needle: {k} is not a permutation of {n}")

    def forward_dev(self, out, x, rows):
        vp = (c_void_p * 5)(*[t.data_ptr() for t in self._vecs])
        fp_ = (c_void_p * 6)(*[t.data_ptr() for t in self._facs])
        check(lib().nd_hadamard_mlp_dev(c_void_p(out.data_ptr()), c_void_p(x.data_ptr()), rows, self.dim, self.na,
                                        self.nb, self.rank, vp, fp_, c_void_p(self._cv.data_ptr()),
                                        c_void_p(self._cu.data_ptr()), c_void_p(self._p[0].data_ptr()),
                                        c_void_p(self._p[1].data_ptr()), _stream()))


class Linear:
    """needle.Linear over a packed matrix (internal/needle/linear.go:11-145),
    on device tensors: x rows × In -> dst rows × Out. With WithInt8Input the
    input rows are first quantised per row (quantInput, int8.go:81-88)."""

    def __init__(self, m, act8=False):
        self.q, self.act8 = m, bool(act8)
        self.In, self.Out = m.In(), m.Out()

    def WithInt8Input(self, on):
        return Linear(self.q, on)

    def Int8Input(self):
        return self.act8

    def _quant_input(self, x, rows):
        import torch

        xq = torch.empty(rows * self.In, dtype=torch.float32, device=x.device)
        fake_quant_dev(xq, x, rows, self.In, self.In)
        return xq

    def Apply(self, dst, x, rows):
        """linear.go:82-95."""
        from . import cq

        if self.act8:
            x = self._quant_input(x, rows)
        cq.gemms_dev([self.q], [dst], x, rows)


def ApplyShared(dsts, x, rows, *ls):
    """ApplyShared (linear.go:97-145): each dsts[k] = ls[k].Apply's result bit
    for bit; the linears that quantise their input share one quantised copy
    of x, and the packed ones of each kind run through one cq.GEMMs."""
    from . import cq

    if len(dsts) != len(ls):
        raise CQPanic(f"needle: ApplyShared of {len(ls)} linears into {len(dsts)} outputs")
    if not ls:
        return
    xq = next((l._quant_input(x, rows) for l in ls if l.act8), None)
    for quant in (False, True):
        sel = [k for k, l in enumerate(ls) if l.act8 == quant]
        if sel:
            cq.gemms_dev([ls[k].q for k in sel], [dsts[k] for k in sel], xq if quant else x, rows)


# ---- caches and memories of any type and length, log probabilities ----------------


# A small call's kernel takes 4 to 8 us, so the checks here are kept to 2 to 4:
# one attribute of a tensor costs 50 to 200 ns.
_TYPES = {}
_torch = _i32 = _f32 = None
_layout = struct.Struct("10q").pack  # nd_cross_layout
_heads_layout = struct.Struct("8q").pack  # nd_heads_layout


def _type(t, what, cache=False):
    """ND_F32.. of a tensor's dtype; ND_I8 and ND_E4M3_PAGES for caches only."""
    global _torch, _i32, _f32
    if _torch is None:
        import torch

        _TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3, torch.float8_e4m3fn: 6})
        _i32, _f32, _torch = torch.int32, torch.float32, torch  # _torch last: other threads look at it
    code = _TYPES.get(t.dtype)
    if code is None or (code >= 3 and not cache):
        raise CQPanic(f"needle: {what} of {t.dtype}")
    return code


def _index(t, what):
    """The index of the GPU a tensor is on."""
    index = t.get_device()
    if index < 0:
        raise CQPanic(f"needle: {what} on {t.device}, not a GPU")
    return index


def _want(t, what, shape, dtype, index, dense=True):
    """Refuses a tensor that the call would read or write out of its bounds."""
    if t.dtype is dtype and t.get_device() == index and t.shape == shape and (not dense or t.is_contiguous()):
        return
    if t.shape != shape:
        raise CQPanic(f"needle: {what} of shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.dtype != dtype:
        raise CQPanic(f"needle: {what} of {t.dtype}, not {dtype}")
    if t.get_device() != index:
        raise CQPanic(f"needle: {what} on {t.device}, not cuda:{index}")
    raise CQPanic(f"needle: {what} that is not contiguous")


_INT = 0x7FFFFFFF  # the calls' sizes are C ints, which ctypes cuts to 32 bits


def _sizes(what, *sizes):
    for n in sizes:
        if not 0 <= n <= _INT:
            raise CQPanic(f"needle: {what} of {n}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(fn, index, *args):
    """fn(*args, the current stream of that GPU), with it current."""
    c = _torch._C
    if index == c._cuda_getDevice():
        rc = fn(*args, c._cuda_getCurrentRawStream(index))
    else:
        with _torch.cuda.device(index):
            rc = fn(*args, c._cuda_getCurrentRawStream(index))
    if rc:
        check(rc)


class PagedKV:
    """Paged key and value caches of many streams (kv_paged, cqhip.h): pools k
    [pages, page_rows, kv_heads, qk] and v [pages, page_rows, kv_heads, vd] of
    float32, float16, bfloat16 or int8 (with scales ks, vs [pages, page_rows,
    kv_heads] float32), or of int8 or float8_e4m3fn with one scale a page and
    head (ks, vs [pages, kv_heads] float32), read through the page table `pages`
    [streams, pages per stream] int32. The tensors stay the caller's: a changed
    table entry or a fork's copied table is seen by the next call. Another
    tensor takes another PagedKV."""

    def __init__(self, k, v, pages, ks=None, vs=None):
        if k.dim() != 4 or v.dim() != 4 or pages.dim() != 2:
            raise CQPanic("needle: a paged cache is [pages, page_rows, kv_heads, width] and its table [streams, pages]")
        self.type, self.index = _type(k, "a cache", cache=True), _index(k, "keys")
        _want(k, "keys", k.shape, k.dtype, self.index)
        _want(v, "values", (*k.shape[:3], v.shape[3]), k.dtype, self.index)
        _want(pages, "page table", pages.shape, _i32, self.index)
        if (self.type >= 3) != (ks is not None) or (ks is None) != (vs is None):
            raise CQPanic("needle: 8-bit caches have scales, float ones none")
        if ks is not None and self.type == 3 and ks.dim() == 2:
            self.type = 5  # a scale a page
        for s, what in ((ks, "key scales"), (vs, "value scales")):
            if s is not None:
                _want(s, what, k.shape[:3] if self.type == 3 else (k.shape[0], k.shape[2]), _f32, self.index)
        self._tensors = k, v, ks, vs, pages
        self.streams, self.kv_heads, self.qk, self.vd = pages.shape[0], k.shape[2], k.shape[3], v.shape[3]
        _sizes("a paged cache", *pages.shape, *k.shape, v.shape[3])
        self.device, self.cap = k.device, min(pages.shape[1] * k.shape[1], _INT)
        self._c = KvPaged(k.data_ptr(), v.data_ptr(), _ptr(ks), _ptr(vs), pages.data_ptr(), self.type, k.shape[2],
                          k.shape[3], v.shape[3], pages.shape[1], k.shape[1], k.shape[0])
        self._ref = ctypes.byref(self._c)

    # Read-only: the calls go by the addresses that _c took.
    k, v, ks, vs, pages = (property(lambda self, i=i: self._tensors[i]) for i in range(5))

    def _acc(self, acc, what, rows):
        cap = acc.shape[-1] if acc.dim() else 0
        _want(acc, what, (self.streams, self.kv_heads, cap), _f32, self.index)
        if cap < rows:
            raise CQPanic(f"needle: {what} of {cap} rows for {rows}")
        return cap

    def append_dev(self, k, v, pos, rows=None, cap=None, acc=None):
        """Rows k [streams, t, kv_heads, qk], v [streams, t, kv_heads, vd]
        (float32, float16, bfloat16; any stream and row strides) appended at
        row pos[b] of stream b, the first rows[b] of them where given; rows
        at or past cap (all that the table holds) are skipped. acc [streams,
        kv_heads, >= cap]: their accumulated weights become 0. With a scale a
        page, a page's scale rises with the rows appended to it, and its codes
        are rounded anew (kv_append_paged_dev, cqhip.h)."""
        shape, code = k.shape, _type(k, "rows")
        t = shape[1] if len(shape) == 4 else 0
        _want(k, "key rows", (self.streams, t, self.kv_heads, self.qk), k.dtype, self.index, dense=False)
        _want(v, "value rows", (self.streams, t, self.kv_heads, self.vd), k.dtype, self.index, dense=False)
        ks, vs = k.stride(), v.stride()
        for x, w, what in ((ks, self.qk, "key rows"), (vs, self.vd, "value rows")):
            if x[3] != 1 or (x[2] != w and self.kv_heads > 1):
                raise CQPanic(f"needle: {what} whose heads are not side by side")
        _want(pos, "positions", (self.streams,), _i32, self.index)
        if rows is not None:
            _want(rows, "row counts", (self.streams,), _i32, self.index)
        if cap is None:
            cap = self.cap
        if t > _INT or not 0 <= cap <= _INT:
            _sizes("append", t, cap)
        acc_cap = self._acc(acc, "weights", cap) if acc is not None else 0
        _call(lib().kv_append_paged_dev, self.index, self._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
              code, self.streams, t, _ptr(rows), pos.data_ptr(), cap, _ptr(acc), acc_cap)

    def read_dev(self, k, v, pos, rows=None):
        """Rows pos[b] + i of stream b's cache as values into k [streams, t,
        kv_heads, qk] and v [streams, t, kv_heads, vd] (float32, float16,
        bfloat16; any stream and row strides), the first rows[b] of them where
        given; rows that the cache does not hold are left as they were."""
        shape, code = k.shape, _type(k, "rows")
        t = shape[1] if len(shape) == 4 else 0
        _want(k, "key rows", (self.streams, t, self.kv_heads, self.qk), k.dtype, self.index, dense=False)
        _want(v, "value rows", (self.streams, t, self.kv_heads, self.vd), k.dtype, self.index, dense=False)
        ks, vs = k.stride(), v.stride()
        for x, w, what in ((ks, self.qk, "key rows"), (vs, self.vd, "value rows")):
            if x[3] != 1 or (x[2] != w and self.kv_heads > 1):
                raise CQPanic(f"needle: {what} whose heads are not side by side")
        _want(pos, "positions", (self.streams,), _i32, self.index)
        if rows is not None:
            _want(rows, "row counts", (self.streams,), _i32, self.index)
        if t > _INT:
            _sizes("a read", t)
        _call(lib().kv_read_paged_dev, self.index, self._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
              code, self.streams, t, _ptr(rows), pos.data_ptr())

    def attend_rows_dev(self, out, q, pos, scale, rows=None, nk_max=None, window=0, sink=0):
        """Causal attention of many rows a stream: row i of q [streams, t,
        heads, qk] and out [streams, t, heads, vd] (one type of float32, float16,
        bfloat16; any stream and row strides) at position pos[b] + i attends the
        cache's rows up to its own, with window > 0 only the last `window` of
        them and the first `sink`; logits q.k / scale. rows [streams]: rows past
        it are left as they were. nk_max (all that the table holds): streams
        whose rows pass it are left as they were."""
        shape, code = q.shape, _type(q, "queries")
        t, heads = (shape[1], shape[2]) if len(shape) == 4 else (0, 0)
        _want(q, "queries", (self.streams, t, heads, self.qk), q.dtype, self.index, dense=False)
        _want(out, "outputs", (self.streams, t, heads, self.vd), q.dtype, self.index, dense=False)
        qs, ys = q.stride(), out.stride()
        if qs[3] != 1 or ys[3] != 1 or (heads > 1 and (qs[2] != self.qk or ys[2] != self.vd)):
            raise CQPanic("needle: queries or outputs whose heads are not side by side")
        _want(pos, "positions", (self.streams,), _i32, self.index)
        if rows is not None:
            _want(rows, "row counts", (self.streams,), _i32, self.index)
        if nk_max is None:
            nk_max = self.cap
        if t > _INT or not 0 <= nk_max <= _INT or not 0 <= window <= _INT or not 0 <= sink <= _INT:
            _sizes("attention", t, nk_max, window, sink)
        _call(lib().kv_attend_rows_paged_dev, self.index, self._ref, out.data_ptr(), ys[0], ys[1], q.data_ptr(), qs[0],
              qs[1], code, self.streams, t, heads, _ptr(rows), pos.data_ptr(), nk_max, window, sink, scale)

    def attend_dev(self, out, q, spans, nk_max, scale, acc=None, acc_out=None):
        """Attention of one token a stream: q [streams, heads, qk] and out
        [streams, heads, vd] of one type (float32, float16, bfloat16), over the
        rows of spans [streams, 4] int32 in [0, nk_max), logits q.k / scale.
        acc_out [streams, kv_heads, >= nk_max]: acc (or 0) plus each row's
        weights; it may be acc."""
        shape, code = q.shape, _type(q, "queries")
        heads = shape[1] if len(shape) == 3 else 0
        _want(q, "queries", (self.streams, heads, self.qk), q.dtype, self.index)
        _want(out, "outputs", (self.streams, heads, self.vd), q.dtype, self.index)
        _want(spans, "spans", (self.streams, 4), _i32, self.index)
        if not 0 <= nk_max <= _INT:
            _sizes("attention over keys", nk_max)
        acc_cap = 0
        if acc_out is not None:
            acc_cap = self._acc(acc_out, "weights", nk_max)
            if acc is not None and self._acc(acc, "weights", nk_max) != acc_cap:
                raise CQPanic(f"needle: weights of {acc.shape[-1]} rows to {acc_cap}")
        elif acc is not None:
            raise CQPanic("needle: weights without an output for them")
        _call(lib().kv_attend_paged_dev, self.index, self._ref, out.data_ptr(), 0, q.data_ptr(), 0, code, self.streams,
              heads, spans.data_ptr(), nk_max, scale, _ptr(acc), _ptr(acc_out), acc_cap)

    def evict_dev(self, dst_pages, acc, acc_out, length, length_out, kept, nk_max, sink=0, recent=0):
        """Each stream's first length[b] (<= nk_max) rows cut to keep =
        kept.shape[2] a key head: the first `sink`, the last `recent`, and the
        others of the largest acc, in order, written to the rows of dst_pages
        [streams, pages] of the same pool, pages that no source row is read
        from.
        kept [streams, kv_heads, keep] int32 gets their numbers, acc_out
        [streams, kv_heads, >= keep] their weights, length_out[b] their count."""
        shape, width = kept.shape, dst_pages.shape[-1] if dst_pages.dim() else 0
        keep = shape[2] if len(shape) == 3 else 0
        _want(kept, "kept rows", (self.streams, self.kv_heads, keep), _i32, self.index)
        _want(dst_pages, "page table", (self.streams, width), _i32, self.index)
        _want(length, "lengths", (self.streams,), _i32, self.index)
        _want(length_out, "lengths", (self.streams,), _i32, self.index)
        _sizes("eviction", nk_max, keep, width, sink, recent)
        acc_cap, out_cap = self._acc(acc, "weights", nk_max), self._acc(acc_out, "weights", keep)
        _call(lib().kv_evict_paged_dev, self.index, self._ref, dst_pages.data_ptr(), width,
              acc.data_ptr(), acc_cap, acc_out.data_ptr(), out_cap, length.data_ptr(), length_out.data_ptr(),
              kept.data_ptr(), self.streams, nk_max, keep, sink, recent)


def cross_attend_dev(out, q, k, v, scale, q_len=None, k_len=None, index=None):
    """Cross-attention to encoder states of other lengths: q [streams, t,
    heads, qk] and out [streams, t, heads, vd] (any stream and row strides)
    over memories k [memories, frames, kv_heads, qk], v [memories, frames,
    kv_heads, vd] (any strides but the last), all of one type (float32,
    float16, bfloat16), logits q.k / scale. q_len [streams]: rows past it are
    left as they were; k_len [memories]: frames past it are not attended;
    index [streams]: the memory each stream reads (beams share one)."""
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != 4 or len(ks) != 4 or len(vs) != 4:
        raise CQPanic("needle: cross-attention of [streams, rows, heads, width]")
    B, t, heads, qk = qs
    M, frames, kv_heads, _ = ks
    vd, code, dtype, dev = vs[3], _type(q, "queries"), q.dtype, _index(q, "queries")
    if max(B, t, M, frames) > _INT:
        _sizes("cross-attention", B, t, M, frames)
    _want(out, "outputs", (B, t, heads, vd), dtype, dev, False)
    _want(k, "keys", (M, frames, kv_heads, qk), dtype, dev, False)
    _want(v, "values", (M, frames, kv_heads, vd), dtype, dev, False)
    qs, ys, ks, vs = q.stride(), out.stride(), k.stride(), v.stride()
    if qs[3] != 1 or ys[3] != 1 or (heads > 1 and (qs[2] != qk or ys[2] != vd)):
        raise CQPanic("needle: queries or outputs whose heads are not side by side")
    if ks[3] != 1 or vs[3] != 1:
        raise CQPanic("needle: memories whose values are not side by side")
    if q_len is not None:
        _want(q_len, "query lengths", (B,), _i32, dev)
    if k_len is not None:
        _want(k_len, "memory lengths", (M,), _i32, dev)
    if index is not None:
        _want(index, "memory index", (B,), _i32, dev)
    _call(lib().nd_cross_attend_dev, dev, out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), code,
          _layout(qs[0], qs[1], ys[0], ys[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2]), B, t, heads, kv_heads, qk, vd, M,
          frames, _ptr(q_len), _ptr(k_len), _ptr(index), scale)


def logprobs_dev(logits, tokens=None, lp=None, ent=None, top=None, top_lp=None):
    """From logits [rows, n] (float32, float16, bfloat16; any row stride), in
    one pass: lp [rows] the log probabilities of tokens [rows] int32 (0 for a
    negative one, a padded row), ent [rows] the entropies, top [rows, k]
    int32 and top_lp [rows, k] the k <= 64 likeliest tokens, the lowest first
    among equals, with their log probabilities."""
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2:
        raise CQPanic(f"needle: logits of shape {tuple(shape)}, not rows of them")
    rows, n = shape
    if rows > _INT or n > _INT:
        _sizes("logits", rows, n)
    code, dev = _type(logits, "logits"), _index(logits, "logits")
    if n > 1 and stride[1] != 1:
        raise CQPanic("needle: logits whose rows are not contiguous")
    k = top.shape[1] if top is not None and top.dim() == 2 else 0
    if tokens is not None:
        _want(tokens, "tokens", (rows,), _i32, dev)
    if lp is not None:
        _want(lp, "log probabilities", (rows,), _f32, dev)
    if ent is not None:
        _want(ent, "entropies", (rows,), _f32, dev)
    if top is not None:
        _want(top, "alternatives", (rows, k), _i32, dev)
    if top_lp is not None:
        _want(top_lp, "alternatives' log probabilities", (rows, k), _f32, dev)
    _call(lib().nd_logprobs_dev, dev, _ptr(lp), _ptr(ent), _ptr(top) if k else None, _ptr(top_lp) if k else None,
          logits.data_ptr(), stride[0], code, rows, n, _ptr(tokens), k)


def qk_norm_rope_dev(q_out, k_out, q, k, q_gain=None, k_gain=None, rope=None, pos=None, rows=None):
    """The norms of the query heads q [streams, t, heads, width] and the key
    heads k [streams, t, kv_heads, width] (one type of float32, float16,
    bfloat16; any stream and row strides) and their rotation in one pass, to
    q_out and k_out, which may be q and k: ZCRMSNorm a head with q_gain, k_gain
    [width] float32 (None: none), then RoPE by row pos[b] + i of rope = (cos, sin),
    tables [positions, width / 2] float32 (None: none). rows [streams]: rows past
    it are left as they were. q and q_out, or k and k_out, may be None."""
    some = q if q is not None else k
    if some is None or (q is None) != (q_out is None) or (k is None) != (k_out is None):
        raise CQPanic("needle: norms without heads or without an output for them")
    shape = some.shape
    if len(shape) != 4:
        raise CQPanic("needle: norms of [streams, rows, heads, width]")
    B, t, heads, width = shape
    code, dtype, dev = _type(some, "heads"), some.dtype, _index(some, "heads")
    kv_heads = 0
    if q is None:
        heads, qs, qo = 0, (0, 0), (0, 0)
    else:
        if q_out.shape != shape or q_out.dtype is not dtype or q_out.get_device() != dev:
            _want(q_out, "normed queries", shape, dtype, dev, False)
        qs, qo = q.stride(), q_out.stride()
        if qs[3] != 1 or qo[3] != 1 or (heads > 1 and (qs[2] != width or qo[2] != width)):
            raise CQPanic("needle: queries whose heads are not side by side")
    if k is None:
        ks = ko = (0, 0)
    else:
        kv_heads = k.shape[2] if k.dim() == 4 else 0
        shape = (B, t, kv_heads, width)
        if k.shape != shape or k.dtype is not dtype or k.get_device() != dev:
            _want(k, "keys", shape, dtype, dev, False)
        if k_out.shape != shape or k_out.dtype is not dtype or k_out.get_device() != dev:
            _want(k_out, "normed keys", shape, dtype, dev, False)
        ks, ko = k.stride(), k_out.stride()
        if ks[3] != 1 or ko[3] != 1 or (kv_heads > 1 and (ks[2] != width or ko[2] != width)):
            raise CQPanic("needle: keys whose heads are not side by side")
    qg = kg = cos = sin = at = None
    if q_gain is not None:
        _want(q_gain, "query gains", (width,), _f32, dev)
        qg = q_gain.data_ptr()
    if k_gain is not None:
        _want(k_gain, "key gains", (width,), _f32, dev)
        kg = k_gain.data_ptr()
    positions = 0
    if rope is not None:
        cos, sin = rope
        positions = cos.shape[0] if cos.dim() == 2 else 0
        shape = (positions, width // 2)
        _want(cos, "cosines", shape, _f32, dev)
        _want(sin, "sines", shape, _f32, dev)
        if pos is None:
            raise CQPanic("needle: RoPE without positions")
        _want(pos, "positions", (B,), _i32, dev)
        cos, sin, at = cos.data_ptr(), sin.data_ptr(), pos.data_ptr()
    if rows is not None:
        _want(rows, "row counts", (B,), _i32, dev)
    if B > _INT or t > _INT or heads > _INT or kv_heads > _INT or width > _INT or positions > _INT:
        _sizes("norms", B, t, heads, kv_heads, width, positions)
    _call(lib().nd_qk_norm_rope_dev, dev, _ptr(q_out), _ptr(k_out), _ptr(q), _ptr(k), code,
          _heads_layout(qs[0], qs[1], ks[0], ks[1], qo[0], qo[1], ko[0], ko[1]), B, t, heads, kv_heads, width, qg, kg, cos, sin,
          positions, at, _ptr(rows))


def verify_drafts_dev(accepted, tokens, target, drafts, draft=None, u=None, u_next=None, drafted=None, temperature=1.0,
                      lp=None):
    """Drafted tokens drafts [streams, t] int32 (the first drafted[b] of them
    where given) verified against the target's logits target [streams, t + 1, n]
    (float32, float16, bfloat16; any stream and row strides) from the random
    numbers u [streams, t] and u_next [streams] float32 in [0, 1); draft
    [streams, t, n]: the logits that they were drawn from (None: each was chosen
    for sure). accepted [streams] int32 gets the count of those kept, tokens
    [streams, t + 1] int32 them, the next token, and -1 behind, lp [streams,
    t + 1] float32 their log probabilities. temperature 0 is greedy, and takes
    no random numbers (nd_verify_drafts_dev, cqhip.h)."""
    shape = target.shape
    if len(shape) != 3 or drafts.dim() != 2:
        raise CQPanic("needle: drafts [streams, t] against logits [streams, t + 1, n]")
    B, t, n = drafts.shape[0], drafts.shape[1], shape[2]
    code, dtype, dev = _type(target, "logits"), target.dtype, _index(target, "logits")
    _want(target, "logits", (B, t + 1, n), dtype, dev, False)
    _want(drafts, "drafts", (B, t), _i32, dev)
    _want(accepted, "accepted counts", (B,), _i32, dev)
    _want(tokens, "tokens", (B, t + 1), _i32, dev)
    ts, ds = target.stride(), (0, 0, 1)
    if draft is not None:
        _want(draft, "the draft's logits", (B, t, n), dtype, dev, False)
        ds = draft.stride()
    if n > 1 and (ts[2] != 1 or ds[2] != 1):
        raise CQPanic("needle: logits whose rows are not contiguous")
    if u is not None:
        _want(u, "random numbers", (B, t), _f32, dev)
    if u_next is not None:
        _want(u_next, "random numbers", (B,), _f32, dev)
    if drafted is not None:
        _want(drafted, "draft counts", (B,), _i32, dev)
    if lp is not None:
        _want(lp, "log probabilities", (B, t + 1), _f32, dev)
    if max(B, t, n) > _INT:
        _sizes("drafts", B, t, n)
    _call(lib().nd_verify_drafts_dev, dev, accepted.data_ptr(), tokens.data_ptr(), _ptr(lp), target.data_ptr(), ts[0],
          ts[1], _ptr(draft), ds[0], ds[1], code, B, t, n, drafts.data_ptr(), _ptr(drafted), _ptr(u), _ptr(u_next),
          temperature)
