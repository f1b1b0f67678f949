"""CPU tests of the batch operators' host side: what the runtime refuses (runtime/batch.h, built
here by itself), the launches it makes, and the Python side's pages and parts."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from skyla_hip import batch as B
from skyla_hip import engine as E

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
RUNTIME = os.path.join(ROOT, "skyla-kernel_amd", "csrc", "runtime")

SHIM = r"""
#include "batch.h"
extern "C" int refuse(const char *name, const uint32_t *spec, const uint32_t *w, const uint32_t *groups,
                      const uint64_t *bytes, char *why) {
  const std::string s = batch::refusal(batch::op_of(name), spec, w, groups, bytes);
  std::strcpy(why, s.c_str());
  return !s.empty();
}
extern "C" int shape(const char *name, const uint32_t *spec, const uint32_t *w, uint32_t rows, uint32_t *groups) {
  const batch::Shape s = batch::shape(batch::op_of(name), spec, w, rows);
  std::copy(s.groups, s.groups + 3, groups);
  return (int)s.threads;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("batch")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", RUNTIME, "-o", str(so),
                    str(src)], check=True)
    return C.CDLL(str(so))


def _refuse(host, name, spec, words, rows, buffers, groups=None):
    u32 = lambda v: (C.c_uint32 * max(1, len(v)))(*[int(x) & 0xFFFFFFFF for x in v])  # noqa: E731
    why = C.create_string_buffer(512)
    bad = host.refuse(name.encode(), u32(spec), u32(words), u32(groups or [1, rows, 1]),
                      (C.c_uint64 * len(buffers))(*buffers), why)
    assert bad == bool(why.value)
    return why.value.decode()


# an arena of 1 MiB; a pool of 8 pages of 32 positions, 2 key heads: f16 keys, 8-bit values
A, W, KV_DIM, SLOTS = 1 << 20, 4096, 256, 256
POOL = SLOTS * KV_DIM * 2 + SLOTS * KV_DIM + SLOTS * KV_DIM // 32 * 2


def _append(**over):
    w = dict(q_off=64, k_off=4096, v_off=6144, o_off=8192, qn=0, kn=128, rope=256, eps=0, mscale=0, n_head=4, n_kv=2,
             qs=512, kvs=256, os=512, kc=0, vc=SLOTS * KV_DIM * 2, ks=0, vs=SLOTS * KV_DIM * 3 // 2, rows=20000,
             table=20100, ts=4, n_seq=3, n_pages=8, log2=5)
    assert not set(over) - set(w)
    return list((w | over).values())


def _attend(**over):
    w = dict(q=64, qs=512, o=4096, os=512, part=8192, kc=0, vc=SLOTS * KV_DIM * 2, ks=0, vs=SLOTS * KV_DIM * 3 // 2,
             n_kv=2, scale=0, n_shared=1, n_own=2, rows=20000, table=20100, ts=4, n_seq=3, n_pages=8, log2=5, wide=0)
    assert not set(over) - set(w)
    return list((w | over).values())


def _logits(**over):
    w = dict(x=64, y=8192, xs=1024, ys=1024, v=1000, ctrl=20000, hist=20100, hs=100, bias=20600, bs=20, mask=20800, ms=32)
    assert not set(over) - set(w)
    return list((w | over).values())


def test_append_words(host):
    ok = lambda rows=4, **k: _refuse(host, "kv_append", [0, 1, 128], _append(**k), rows, [W, A, A, POOL, POOL])  # noqa: E731
    assert ok() == "" and ok(rows=0) == "" and ok(o_off=64) == ""
    for bad in (dict(q_off=A // 4 - 100), dict(k_off=A // 4), dict(v_off=2**32 - 1), dict(o_off=2**32 - 4), dict(qn=W // 4),
                dict(rope=W // 4 - 63), dict(n_head=0), dict(n_kv=0), dict(n_head=2**31), dict(qs=100), dict(kvs=0),
                dict(kc=8), dict(kc=3), dict(vc=SLOTS * KV_DIM * 2 + 8), dict(vs=SLOTS * KV_DIM * 3 // 2 + 4), dict(rows=20001),
                dict(rows=A // 4), dict(table=A // 4 - 11), dict(ts=0), dict(n_seq=0), dict(n_seq=2**30), dict(n_pages=0),
                dict(n_pages=9), dict(log2=3), dict(log2=13), dict(log2=31), dict(log2=40), dict(o_off=512), dict(o_off=4096),
                dict(o_off=6144 - 512), dict(o_off=19600), dict(o_off=64, os=516)):
        assert ok(**bad), bad
    assert ok(rows=65536) and "rows" in ok(rows=65536)
    assert _refuse(host, "kv_append", [0, 1, 128], _append(), 4, [W, A, A, POOL, POOL], groups=[2, 4, 1])


def test_attention_words(host):
    ok = lambda rows=4, **k: _refuse(host, "attention_paged", [2, 0, 1, 128], _attend(**k), rows, [A, A, POOL, POOL, POOL])  # noqa: E731
    assert ok() == "" and ok(o=64) == "" and ok(n_shared=0) == ""
    for bad in (dict(q=A // 4), dict(q=65), dict(qs=510), dict(o=4097), dict(part=8193), dict(part=A // 4 - 100), dict(part=4096),
                dict(part=512), dict(part=19000), dict(n_own=0), dict(n_own=1025), dict(n_shared=1024), dict(n_shared=2**32 - 1),
                dict(n_kv=0), dict(n_kv=3), dict(n_kv=2**31), dict(kc=8), dict(ks=2, n_pages=9), dict(vs=2), dict(table=2**32 - 1),
                dict(n_seq=0), dict(ts=9), dict(ts=2**31), dict(log2=2), dict(wide=2), dict(o=68), dict(os=516, o=64), dict(o=20000), dict(o=19900)):
        assert ok(**bad), bad
    assert ok(rows=65535)  # the partials end past the arena
    # 8-bit keys: the key rows and their scales in bytes and halves
    q8 = lambda **k: _refuse(host, "attention_paged", [2, 1, 1, 128], _attend(vc=SLOTS * KV_DIM, ks=SLOTS * KV_DIM,  # noqa: E731
                                                                             **({"vs": SLOTS * KV_DIM + SLOTS * KV_DIM // 32} | k)),
                             4, [A, A, POOL, POOL, POOL])
    assert q8() == "" and q8(vs=POOL // 2 - 4) and q8(vs=SLOTS * KV_DIM + 2)


def test_merge_words(host):
    base = dict(part=8192, o=4096, os=512, n_head=4, n_shared=1, n_own=2, rows=20000, ts=4, n_seq=3, log2=5)
    ok = lambda rows=4, **k: _refuse(host, "attention_paged_merge", [128], list((base | k).values()), rows, [A, A])  # noqa: E731
    assert ok() == ""
    for bad in (dict(part=A // 4 - 6000), dict(part=1 << 31), dict(o=8190), dict(os=256), dict(n_head=0), dict(n_own=0),
                dict(n_shared=1024), dict(n_shared=0, n_own=1), dict(rows=2**31), dict(log2=0), dict(o=19998)):
        assert ok(**bad), bad


def test_logits_words(host):
    ok = lambda rows=4, **k: _refuse(host, "logits_adjust", [], _logits(**k), rows, [A, A])  # noqa: E731
    assert ok() == "" and ok(y=64) == "" and ok(hs=0, bs=0, ms=0, hist=2**32 - 4, bias=2**32 - 4, mask=2**32 - 4) == ""
    for bad in (dict(x=65), dict(xs=1002), dict(x=A // 4), dict(y=1024), dict(y=64, ys=1028), dict(v=0), dict(v=1025),
                dict(ctrl=A // 4 - 28), dict(hist=A // 4 - 100), dict(hs=101), dict(bs=21), dict(ms=31), dict(mask=A // 4 - 32),
                dict(y=16500), dict(bias=11000)):
        assert ok(**bad), bad


def test_unknown_names_and_launches(host):
    assert _refuse(host, "matvec_q4k", [], [], 1, [16]) == ""   # not a batch operator: its words are the caller's
    g = (C.c_uint32 * 3)()
    u32 = lambda v: (C.c_uint32 * len(v))(*v)  # noqa: E731
    for rows in (1, 7, 128, 2048):
        host.shape(b"kv_append", u32([0, 1, 128]), u32(_append()), rows, g)
        assert g[0] * g[1] >= 1 and g[2] == 1
        for v in (1, 1000, 4097, 151936):
            t = host.shape(b"logits_adjust", u32([0]), u32(_logits(v=v)), rows, g)
            assert g[1] == rows and g[2] == 1 and g[0] == -(-v // (16 * t))


def test_pages_and_parts():
    for bad in (dict(page=8), dict(page=24), dict(page=8192), dict(n_pages=0), dict(n_seq=0), dict(seq_pages=0), dict(kv_dim=100)):
        with pytest.raises(ValueError):
            B.Paged(**(dict(precision=E.KvPrecision.F16, page=16, n_pages=4, n_seq=1, seq_pages=2, kv_dim=256) | bad))
    p = B.Paged(E.KvPrecision.F16_KEYS_Q8_VALUES, 32, 8, 3, 4, 256)
    assert p.bytes() == POOL and p.page_log2 == 5
    for rows in (1, 3, 128, 1000):
        for shared in (0, 1, 64, 100000):
            for own in (1, 65, 20000):
                for n_kv, rep in ((1, 1), (8, 4), (4, 8)):
                    s, o, wide = B.splits(rows, n_kv, rep, shared, own)
                    assert not wide or shared
                    assert (s == 0) == (shared == 0) and o >= 1 and s + o <= B.MAX_PARTS
                    assert s <= max(1, -(-shared // 64)) and o <= max(1, -(-own // 64))
    assert B.part_size(3, 8, (2, 5)) == 3 * 8 * 7 * 130
    assert np.all([B.PAGE_SIZES[i] == 16 << i for i in range(9)])
