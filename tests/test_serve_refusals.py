"""Misuse of the serving operators' entry points, refused before any device
call (no GPU): sizes, types, widths, alignment, missing operands."""

import ctypes

import pytest

from go_whistle_amd import _lib, needle
from go_whistle_amd._lib import CQDeviceError, CQPanic, CrossLayout, KvPaged, check, lib

P = 256  # a pointer that is never dereferenced: the checks come first


def cache(**kw):
    c = KvPaged(P, P, None, None, P, 1, 2, 64, 64, 4, 16, 8)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


BAD_CACHES = [(dict(type=4), CQPanic), (dict(type=-1), CQPanic), (dict(kv_heads=0), CQPanic), (dict(qk=40), CQDeviceError),
              (dict(vd=272), CQDeviceError), (dict(qk=0), CQDeviceError), (dict(page_rows=12), CQPanic),
              (dict(page_rows=0), CQPanic), (dict(pool_pages=0), CQPanic), (dict(page_stride=3), CQPanic),
              (dict(page_stride=-1), CQPanic), (dict(k=None), CQPanic), (dict(v=None), CQPanic),
              (dict(pages=None), CQPanic), (dict(type=3), CQPanic), (dict(k=P + 8), CQPanic), (dict(v=P + 2), CQPanic),
              (dict(pool_pages=1 << 30, page_rows=4, page_stride=64), CQDeviceError)]


def append(c=None, k=P, v=P, typ=0, batch=2, t=3, pos=P, cap=64, acc=None, acc_cap=0):
    check(lib().kv_append_paged_dev(c or cache(), k, 0, 0, v, 0, 0, typ, batch, t, None, pos, cap, acc, acc_cap, None))


def attend(c=None, out=P, q=P, typ=0, batch=2, heads=4, spans=P, nk=64, scale=8.0, acc=None, acc_out=None, acc_cap=0):
    check(lib().kv_attend_paged_dev(c or cache(), out, 0, q, 0, typ, batch, heads, spans, nk, scale, acc, acc_out,
                                    acc_cap, None))


def evict(c=None, dst=P, stride=4, acc=P, acc_cap=64, out=2 * P, out_cap=64, ln=P, ln_out=P, kept=P, batch=2, nk=64,
          keep=32, sink=4, recent=4):
    check(lib().kv_evict_paged_dev(c or cache(), dst, stride, acc, acc_cap, out, out_cap, ln, ln_out, kept, batch, nk,
                                   keep, sink, recent, None))


def cross(out=P, q=P, k=P, v=P, typ=1, layout=None, batch=2, t=3, heads=4, kv_heads=2, qk=64, vd=64, memories=2,
          frames=10, scale=8.0):
    y = ctypes.byref(layout) if layout is not None else None
    check(lib().nd_cross_attend_dev(out, q, k, v, typ, y, batch, t, heads, kv_heads, qk, vd, memories, frames, None,
                                    None, None, scale, None))


def logprobs(lp=P, ent=P, ti=P, tl=P, x=P, stride=100, typ=0, rows=2, n=100, tok=P, top=5):
    check(lib().nd_logprobs_dev(lp, ent, ti, tl, x, stride, typ, rows, n, tok, top, None))


@pytest.mark.parametrize("call", [append, attend, evict])
@pytest.mark.parametrize("edit,err", BAD_CACHES)
def test_bad_caches(call, edit, err):
    with pytest.raises(err):
        call(c=cache(**edit))


@pytest.mark.parametrize("call,kw", [
    (append, dict(batch=-1)), (append, dict(t=-1)), (append, dict(cap=-1)), (append, dict(typ=3)),
    (append, dict(typ=-1)), (append, dict(k=None)), (append, dict(v=None)), (append, dict(pos=None)),
    (append, dict(cap=65)), (append, dict(acc=P, acc_cap=63)), (append, dict(k=P + 2)),
    (append, dict(typ=1, v=P + 1)),
    (attend, dict(batch=-1)), (attend, dict(nk=-1)), (attend, dict(nk=65)), (attend, dict(typ=3)),
    (attend, dict(heads=3)), (attend, dict(heads=0)), (attend, dict(scale=0.0)), (attend, dict(scale=-1.0)), (cross, dict(scale=-1.0)),
    (attend, dict(scale=1e-40)), (cross, dict(scale=1e-40)), (attend, dict(scale=float("nan"))),
    (attend, dict(scale=float("inf"))), (attend, dict(out=None)), (attend, dict(q=None)), (attend, dict(spans=None)),
    (attend, dict(acc_out=P, acc_cap=63)), (attend, dict(q=P + 2)), (attend, dict(typ=2, out=P + 1)),
    (evict, dict(batch=-1)), (evict, dict(nk=-1)), (evict, dict(keep=-1)), (evict, dict(sink=-1)),
    (evict, dict(recent=-1)), (evict, dict(sink=20, recent=13)), (evict, dict(stride=1)), (evict, dict(acc_cap=63)),
    (evict, dict(out_cap=31)), (evict, dict(dst=None)), (evict, dict(acc=None)), (evict, dict(out=None)),
    (evict, dict(ln=None)), (evict, dict(ln_out=None)), (evict, dict(kept=None)), (evict, dict(out=P)),
    (cross, dict(batch=-1)), (cross, dict(t=-1)), (cross, dict(memories=-1)), (cross, dict(frames=-1)),
    (cross, dict(typ=3)), (cross, dict(heads=3)), (cross, dict(kv_heads=0)), (cross, dict(scale=0.0)),
    (cross, dict(out=None)), (cross, dict(q=None)), (cross, dict(k=None)), (cross, dict(v=None)), (cross, dict(k=P + 2)),
    (cross, dict(q=P + 1)), (cross, dict(layout=CrossLayout(768, 256, 768, 256, 1280, 132, 64, 1280, 128, 64))),
    (logprobs, dict(rows=-1)), (logprobs, dict(n=0)), (logprobs, dict(top=-1)), (logprobs, dict(n=4)),
    (logprobs, dict(stride=-1)), (logprobs, dict(typ=3)), (logprobs, dict(tok=None)), (logprobs, dict(ti=None)),
    (logprobs, dict(tl=None)), (logprobs, dict(x=None)), (logprobs, dict(x=P + 2)),
])
def test_misuse(call, kw):
    with pytest.raises(CQPanic):
        call(**kw)


@pytest.mark.parametrize("call,kw", [
    (cross, dict(qk=40)), (cross, dict(vd=264)), (logprobs, dict(top=65)), (logprobs, dict(n=(1 << 30) + 1)),
    (attend, dict(heads=4096)), (append, dict(batch=1 << 20, t=64)),
])
def test_unsupported(call, kw):
    with pytest.raises(CQDeviceError):
        call(**kw)


@pytest.mark.parametrize("call,kw", [
    (append, dict(batch=0)), (append, dict(t=0)), (append, dict(cap=0)), (attend, dict(batch=0)), (evict, dict(batch=0)),
    (cross, dict(batch=0)), (cross, dict(t=0)), (logprobs, dict(rows=0)), (logprobs, dict(lp=None, ent=None, ti=None, tl=None)),
])
def test_nothing_to_do(call, kw):
    call(**kw)


def test_wrappers_refuse_host_tensors_and_shapes():
    import torch

    k = torch.zeros(4, 16, 2, 64)
    pages = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(CQPanic):
        needle.PagedKV(k, k, pages)  # host memory
    with pytest.raises(CQPanic):
        needle.PagedKV(k[0], k, pages)
    with pytest.raises(CQPanic):
        needle.logprobs_dev(torch.zeros(3, 5))
    with pytest.raises(CQPanic):
        needle.logprobs_dev(torch.zeros(5))
    q = torch.zeros(2, 3, 4, 64)
    with pytest.raises(CQPanic):
        needle.cross_attend_dev(q, q, q, q, 8.0)
    with pytest.raises(CQPanic):
        needle.cross_attend_dev(q, q[0], q, q, 8.0)
    assert _lib.SIGNATURES["kv_attend_paged_dev"]


@pytest.mark.parametrize("call,kw", [
    (evict, dict(c=cache(pages=3 * P), dst=3 * P)),  # onto the pages that are read
    (evict, dict(out=P + 1020)), (evict, dict(acc=P + 1020, out=P)),  # weights in part onto themselves
    (attend, dict(acc=P, acc_out=P + 4, acc_cap=64)), (attend, dict(acc=P + 4, acc_out=P, acc_cap=64)),
    (cross, dict(layout=CrossLayout(768, 256, 0, 256, 1280, 128, 64, 1280, 128, 64))),  # outputs of one place
    (cross, dict(layout=CrossLayout(768, 256, 768, 0, 1280, 128, 64, 1280, 128, 64))),
])
def test_outputs_that_would_race(call, kw):
    with pytest.raises(CQPanic, match="onto|one place"):
        call(**kw)


def layout(out_stream, out_row):
    return CrossLayout(768, 256, out_stream, out_row, 1280, 128, 64, 1280, 128, 64)


def spread(batch, t, out_stream, out_row, width=256):
    """Whether batch x t rows of `width` elements share none, by counting."""
    seen = set()
    for b in range(batch):
        for i in range(t):
            at = b * out_stream + i * out_row
            row = set(range(at, at + width))
            if seen & row:
                return False
            seen |= row
    return True


@pytest.mark.parametrize("batch,t", [(1, 1), (1, 3), (2, 1), (2, 3), (3, 2), (4, 5)])
def test_cross_attention_outputs_lie_apart(batch, t):
    # heads * vd = 256; rows that lie apart get as far as the next check, of the memories' alignment
    for out_stream in (0, 1, 255, 256, 257, 300, 511, 512, 600, 767, 768, 1000, 1024, 1279, 1280, 1536, -256, -700, 1 << 40):
        for out_row in (0, 1, 255, 256, 257, 400, 512, 513, 768, 1024, 1300, -256, -512, 1 << 41):
            y = layout(out_stream, out_row)
            if spread(batch, t, out_stream, out_row):
                with pytest.raises(CQPanic, match="aligned to 16 bytes"):
                    cross(batch=batch, t=t, layout=y, k=P + 2)
            else:
                with pytest.raises(CQPanic, match="one place"):
                    cross(batch=batch, t=t, layout=y)


def test_outputs_of_ragged_rows_may_be_packed():
    # rows of 256: with lengths only the first rows of two streams, and two rows of one, are known to be written
    for out_stream, out_row, ok in ((300, 256, True), (256, 600, True), (255, 256, False), (0, 256, False), (768, 255, False)):
        y = layout(out_stream, out_row)
        with pytest.raises(CQPanic, match="aligned to 16 bytes" if ok else "one place"):
            check(lib().nd_cross_attend_dev(P, P, P + 2, P, 1, ctypes.byref(y), 3, 3, 4, 2, 64, 64, 2, 10, P, None, None,
                                            8.0, None))


def test_attention_outputs_lie_apart():
    def strided(stride, batch=2):
        check(lib().kv_attend_paged_dev(cache(), P, stride, P, 0, 0, batch, 4, P, 64, 8.0, P, P + 4, 64, None))

    for stride in (1, 64, 255, -255):  # 4 heads of 64
        with pytest.raises(CQPanic, match="one place"):
            strided(stride)
    for stride, batch in ((0, 2), (256, 2), (257, 2), (-256, 2), (1, 1)):
        with pytest.raises(CQPanic, match="onto"):  # the next check
            strided(stride, batch)


@pytest.mark.parametrize("batch,t", [((1 << 31) - 1, (1 << 31) - 1), (1 << 20, 1 << 10)])
def test_more_outputs_than_a_launch(batch, t):
    with pytest.raises(CQDeviceError):
        cross(batch=batch, t=t, layout=layout(257, 258))


@pytest.mark.parametrize("shift", [-4, 4])
def test_lengths_in_part_onto_themselves(shift):
    # a copy would read one stream's new length as another's old one
    with pytest.raises(CQPanic, match="onto a part"):
        evict(out=64 * P, ln=4 * P, ln_out=4 * P + shift)
    for ln_out in (4 * P, 4 * P + 2 * shift):  # the next check
        with pytest.raises(CQPanic, match="own pages"):
            evict(c=cache(pages=3 * P), dst=3 * P, out=64 * P, ln=4 * P, ln_out=ln_out)


@pytest.mark.parametrize("name", ["k_stream", "v_stream", "k_row", "v_row", "k_head", "v_head"])
def test_strides_of_single_memories_frames_and_heads(name):
    # a stride that leads nowhere may be anything, as torch's strides of dimensions of 1 are
    y = CrossLayout(256, 256, 256, 256, 1280, 128, 64, 1280, 128, 64)
    setattr(y, name, 63)
    single = {"stream": dict(memories=1), "row": dict(frames=1), "head": dict(kv_heads=1)}[name.split("_")[1]]
    with pytest.raises(CQPanic, match="aligned to their type"):  # the next check
        cross(layout=y, batch=1, t=1, q=P + 1, **single)
    with pytest.raises(CQPanic, match="aligned to 16 bytes"):
        cross(layout=y, batch=1, t=1, q=P + 1)
