"""What the launchers of the paged KV cache's operators refuse, and what they accept, without a GPU: the launch arguments of a dry run (all
checks, nothing launched) with made-up addresses."""
import ctypes as C
import struct

import pytest

from conftest import load_pkg

rt = load_pkg().runtime
ARG, FEATURE, SHAPE, ALIGN, SIZE = -303, -108, -109, -203, -206


class LaunchStream(C.Structure):      # csrc/common.cuh, with LaunchArgs
    _fields_ = [("s", C.c_void_p), ("in_order", C.c_bool), ("dry", C.c_bool)]


class LaunchArgs(C.Structure):
    _fields_ = [("stream", LaunchStream), ("binding_count", C.c_uint32), ("ptr", C.c_uint64 * 16),
                ("range", C.c_uint64 * 16), ("push", C.c_uint32 * 32), ("grid", C.c_uint32 * 3), ("status", C.c_void_p), ("sm_count", C.c_int),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64), ("side", C.c_void_p), ("add_e", C.c_void_p), ("add_out", C.c_void_p)]


def bits(v):
    return struct.unpack("<I", struct.pack("<f", v))[0]


def call(symbol, push, ranges, ptr=None):
    fn = getattr(rt.load_library(), symbol)
    fn.restype, fn.argtypes = C.c_int, [C.POINTER(LaunchArgs)]
    a = LaunchArgs(binding_count=len(ranges), sm_count=148)
    a.stream.dry = True
    for i, n in enumerate(ranges):
        a.ptr[i], a.range[i] = (i + 1) << 40, n
    for i, p in (ptr or {}).items():
        a.ptr[i] = p
    for i, w in enumerate(push):
        a.push[i] = w
    return fn(C.byref(a))


# 3 sequences, 5 rows, 8 heads of 128 over 2 KV heads, 12 pages of 16, 4 pages a sequence
D, H, HKV, SEQS, ROWS, PAGE, PAGES, STRIDE = 128, 8, 2, 3, 5, 16, 12, 4
CACHE = PAGES * PAGE * HKV * D * 2
ATTN = dict(D=D, H=H, Hkv=HKV, n_seqs=SEQS, rows=ROWS, max_q=3, max_kv=50, page=PAGE, pages=PAGES, stride=STRIDE, c_ps=PAGE * HKV * D, c_ts=HKV * D, c_hs=D,
            q_s=H * D, dst_s=H * D, f16=0, scale=bits(0.1), softcap=0, last=0, node=1)
ATTN_RANGES = [ROWS * H * D * 2, CACHE, CACHE, SEQS * STRIDE * 4, (SEQS + 1) * 4, SEQS * 4, ROWS * H * D * 4, 1 << 22, 8]
PREFIX_RANGES = ATTN_RANGES + [4 + 4 * 7]
APPEND = dict(D=D, H=H, Hkv=HKV, n_seqs=SEQS, rows=ROWS, page=PAGE, pages=PAGES, stride=STRIDE, c_ps=PAGE * HKV * D, c_ts=HKV * D, c_hs=D, q_s=H * D,
              k_s=HKV * D, v_s=HKV * D, o_s=H * D, n_dims=D, neox=0, flags=3, theta=bits(0.9), freq=bits(1.0), ext=0, attn=bits(1.0), corr0=0, corr1=0, node=1)
APPEND_RANGES = [ROWS * H * D * 4, ROWS * HKV * D * 4, ROWS * HKV * D * 4, SEQS * STRIDE * 4, (SEQS + 1) * 4, SEQS * 4, ROWS * 4, D * 2, ROWS * H * D * 2, CACHE,
                 CACHE, 8]


def attn(ranges=None, ptr=None, **kw):
    return call("_ZN3amv17launch_paged_attnERKNS_10LaunchArgsE", {**ATTN, **kw}.values(), ranges or ATTN_RANGES, ptr)


def prefix(ranges=None, ptr=None, **kw):
    return call("_ZN3amv24launch_paged_prefix_attnERKNS_10LaunchArgsE", {**ATTN, "last": 100, **kw}.values(), ranges or PREFIX_RANGES, ptr)


def append(ranges=None, ptr=None, **kw):
    return call("_ZN3amv19launch_paged_appendERKNS_10LaunchArgsE", {**APPEND, **kw}.values(), ranges or APPEND_RANGES, ptr)


def accepted(rc):
    """Past every check: a machine without a driver has no encoder of tensor maps, or nothing to ask for the last launch's error."""
    return rc not in (ARG, FEATURE, SHAPE, ALIGN, SIZE)


def less(ranges, i, by=1):
    return [n - by if j == i else n for j, n in enumerate(ranges)]


def test_what_is_right_is_accepted():
    assert accepted(attn()) and accepted(prefix()) and accepted(append())
    assert accepted(attn(last=7)) and accepted(attn(softcap=bits(30.0))) and accepted(attn(scale=bits(-0.1)))
    assert accepted(attn(ranges=less(ATTN_RANGES, 6, ROWS * H * D * 2), f16=1))
    assert accepted(attn(c_ps=PAGE * HKV * D, c_ts=D, c_hs=PAGE * D))                # a head's tokens beside one another
    assert accepted(append(c_ps=PAGE * HKV * D, c_ts=D, c_hs=PAGE * D))
    assert accepted(append(n_dims=0)) and accepted(append(n_dims=50, neox=1))
    assert accepted(append(flags=0, ranges=APPEND_RANGES[:6] + [4, 4] + APPEND_RANGES[8:], ptr={6: 6 << 40, 7: 6 << 40}))
    assert accepted(append(page=12, c_ps=12 * HKV * D))                               # a page size of any kind
    # q, k and v as column ranges of one product
    w = (H + 2 * HKV) * D
    base, n = 1 << 41, ROWS * w * 4
    assert accepted(append(q_s=w, k_s=w, v_s=w, ranges=[n, n - H * D * 4, n - (H + HKV) * D * 4] + APPEND_RANGES[3:],
                           ptr={0: base, 1: base + H * D * 4, 2: base + (H + HKV) * D * 4}))


@pytest.mark.parametrize("field", ["D", "H", "Hkv", "n_seqs", "rows", "page", "pages", "stride"])
def test_zero_sizes(field):
    assert attn(**{field: 0}) == ARG and prefix(**{field: 0}) == ARG and append(**{field: 0}) == ARG
    if field == "rows":
        assert attn(max_q=0) == ARG and attn(max_kv=0) == ARG and prefix(last=0) == ARG


@pytest.mark.parametrize("change,code", [
    (dict(H=7), ARG), (dict(page=24), ARG), (dict(f16=2), ARG), (dict(softcap=bits(-1.0)), ARG), (dict(softcap=bits(float("nan"))), ARG),
    (dict(scale=bits(float("nan"))), ARG), (dict(D=96), FEATURE), (dict(D=512), FEATURE), (dict(page=8), FEATURE), (dict(page=2048), FEATURE),
    (dict(n_seqs=4096), SHAPE), (dict(H=131072, Hkv=131072), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(max_kv=0x7FFFFFFF), SHAPE),
    (dict(stride=1 << 28), SHAPE), (dict(dst_s=H * D - 8), SHAPE), (dict(c_ps=4100), ALIGN), (dict(c_ts=260), ALIGN), (dict(c_hs=130), ALIGN),
    (dict(q_s=1028), ALIGN), (dict(dst_s=1026), ALIGN), (dict(dst_s=1028, f16=1), ALIGN)])
def test_attention_sizes(change, code):
    assert attn(**change) == code and prefix(**change) == code


@pytest.mark.parametrize("binding", range(9))
def test_attention_buffers(binding):
    if binding != 7:
        assert attn(ranges=less(ATTN_RANGES, binding)) == SIZE and prefix(ranges=less(PREFIX_RANGES, binding)) == SIZE
    off = 8 if binding in (0, 1, 2, 6, 7) else 2
    assert attn(ptr={binding: ((binding + 1) << 40) + off}) == ALIGN and prefix(ptr={binding: ((binding + 1) << 40) + off}) == ALIGN
    for written in (6, 7, 8):
        if written != binding:      # what is written meets nothing else
            at = ((written + 1) << 40) + ATTN_RANGES[written] - 16 if written != 8 else 9 << 40
            assert attn(ptr={binding: at}) == ARG, written


def test_prefix_buffers():
    assert prefix(ranges=less(PREFIX_RANGES, 9)) == SIZE and prefix(ptr={9: (10 << 40) + 2}) == ALIGN
    assert prefix(ptr={9: 8 << 40}) == ARG and prefix(last=0x7FFFFFFF) == SHAPE
    assert prefix(last=113) == SIZE
    own = ROWS * H * (D + 4) * 4      # the rows' results over their own keys
    own = (own + 255) // 256 * 256
    assert prefix(ranges=PREFIX_RANGES[:7] + [own - 16] + PREFIX_RANGES[8:]) == SIZE and accepted(prefix(ranges=PREFIX_RANGES[:7] + [own] + PREFIX_RANGES[8:]))


def test_a_line_too_long_is_refused():
    """Work that 32 bits do not number: 4095 sequences of a million rows' announcement and as many keys."""
    n, stride = 4095, 1 << 17
    ranges = [(1 << 20) * H * D * 2, CACHE, CACHE, n * stride * 4, (n + 1) * 4, n * 4, (1 << 20) * H * D * 4, 1 << 22, 8]
    assert attn(n_seqs=n, rows=1 << 20, max_q=1 << 20, max_kv=1 << 20, stride=stride, ranges=ranges) == SHAPE


@pytest.mark.parametrize("change,code", [
    (dict(neox=2), ARG), (dict(flags=4), ARG), (dict(n_dims=D + 2), ARG), (dict(n_dims=5), ARG), (dict(D=264, n_dims=64), FEATURE),
    (dict(D=100, n_dims=64), FEATURE), (dict(H=65536), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(stride=1 << 28), SHAPE), (dict(q_s=1026), ALIGN),
    (dict(k_s=258), ALIGN), (dict(v_s=258), ALIGN), (dict(c_ps=4100), ALIGN), (dict(c_ts=260), ALIGN), (dict(c_hs=130), ALIGN), (dict(o_s=1028), ALIGN),
    (dict(o_s=H * D - 8), SHAPE), (dict(c_hs=D - 8), SHAPE), (dict(c_ts=D), SHAPE), (dict(c_ps=HKV * D), SHAPE), (dict(c_ps=0), SHAPE)])
def test_append_sizes(change, code):
    assert append(**change) == code


@pytest.mark.parametrize("binding", range(12))
def test_append_buffers(binding):
    assert append(ranges=less(APPEND_RANGES, binding)) == SIZE
    off = 8 if binding in (0, 1, 2, 8, 9, 10) else 2
    assert append(ptr={binding: ((binding + 1) << 40) + off}) == ALIGN
    for written in (8, 9, 10, 11):
        if written != binding:
            at = ((written + 1) << 40) + APPEND_RANGES[written] - 16 if written != 11 else 12 << 40
            assert append(ptr={binding: at}) == ARG, written
