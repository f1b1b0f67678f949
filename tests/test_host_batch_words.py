"""CPU tests of the batch operators' host side with the buffers' places: overlaps that are refused
whichever binding they go through, and none that are not there."""
import ctypes as C
import subprocess

import pytest

from test_host_batch import A, KV_DIM, POOL, RUNTIME, SLOTS, W, _append, _attend, _logits

SHIM = r"""
#include "batch.h"
extern "C" int refuse(const char *name, const uint32_t *spec, const uint32_t *w, const uint32_t *groups,
                      const uint64_t *bytes, const uint64_t *at, char *why) {
  const std::string s = batch::refusal(batch::op_of(name), spec, w, groups, bytes, at);
  std::strcpy(why, s.c_str());
  return !s.empty();
}
"""


def u32(v):
    return (C.c_uint32 * max(1, len(v)))(*[int(x) & 0xFFFFFFFF for x in v])


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("words")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", RUNTIME, "-o", str(so),
                    str(src)], check=True)
    return C.CDLL(str(so))


def _refuse(host, name, spec, words, bound, rows=4):
    """`bound`: (place, bytes) of each buffer."""
    why = C.create_string_buffer(512)
    u64 = lambda v: (C.c_uint64 * len(v))(*v)  # noqa: E731
    host.refuse(name.encode(), u32(spec), u32(words), u32([1, rows, 1]), u64([b for _, b in bound]),
                u64([p for p, _ in bound]), why)
    return why.value.decode()


ARENA, TABLES, POOLS, WORDS = (1 << 30, A), (1 << 32, W), (1 << 33, POOL), (1 << 34, A)


def test_append_overlaps_by_place(host):
    ok = lambda bound, **k: _refuse(host, "kv_append", [0, 1, 128], _append(**k), bound)  # noqa: E731
    apart = [TABLES, ARENA, ARENA, POOLS, POOLS]
    assert ok(apart) == "" and ok(apart, o_off=64) == ""
    # the tables in the arena: the output over them is refused, beside them it is not
    inside = [(ARENA[0] + 4 * 30000, W), *apart[1:]]
    assert ok(inside) == "" and ok(inside, qn=0, o_off=30000 - 4 * 512) == ""
    for name, over in (("q's norm weights", dict(qn=0, kn=512, o_off=30000 - 4 * 512 + 4)),
                       ("k's norm weights", dict(qn=512, kn=0, o_off=30000 - 4 * 512 + 4)),
                       ("frequencies", dict(qn=512, kn=640, rope=0, o_off=30000 - 4 * 512 + 4))):
        assert name in ok(inside, **over)
    same = [ARENA, ARENA, ARENA, POOLS, POOLS]
    assert ok(same, qn=22000, kn=22128, rope=22256) == ""
    assert "norm weights" in ok(same, qn=8192, kn=22128, rope=22256)
    # a pool in the arena
    pool = (ARENA[0] + 4 * 50000, POOL)
    assert ok([TABLES, ARENA, ARENA, pool, pool]) == ""
    for words in (dict(o_off=50000 - 4), dict(q_off=50000 - 4, o_off=60000), dict(k_off=50000), dict(v_off=52000), dict(rows=49988),
                  dict(table=50000 - 11)):
        assert "overlap" in ok([TABLES, ARENA, ARENA, pool, pool], **words), words
    # the control words
    over = dict(qn=22000, kn=22128, rope=22256, q_off=40000, o_off=4)
    assert "control words" in ok(same, **over) and ok([ARENA, ARENA, WORDS, POOLS, POOLS], **over) == ""
    # equal offsets in buffers of their own are no overlap
    assert ok(apart[:2] + [WORDS] + apart[3:], rows=8192, table=8200) == ""
    assert ok([TABLES, ARENA, (WORDS[0], 16), POOLS, POOLS])  # no room for the control words
    # 8-bit values in a buffer of their own, at the keys' offsets
    assert ok([TABLES, ARENA, ARENA, POOLS, (1 << 35, POOL)], vc=0, vs=SLOTS * KV_DIM) == ""
    assert "overlap" in ok(apart, vc=0, vs=SLOTS * KV_DIM)


def test_attention_overlaps_by_place(host):
    ok = lambda bound, **k: _refuse(host, "attention_paged", [2, 0, 1, 128], _attend(**k), bound)  # noqa: E731
    apart = [ARENA, ARENA, POOLS, POOLS, POOLS]
    assert ok(apart) == "" and ok(apart, o=64) == ""
    pool = (ARENA[0] + 4 * 50000, POOL)
    inside = [ARENA, ARENA, pool, pool, pool]
    assert ok(inside) == "" and ok(inside, q=50000) == ""  # read by both
    assert "overlap" in ok(inside, o=50000 - 2) and "overlap" in ok(inside, part=50000 - 2)
    assert "control words" in ok(apart, o=0, q=40000) and "control words" in ok(apart, part=4, q=40000, o=44000, n_shared=0)
    words = [ARENA, WORDS, POOLS, POOLS, POOLS]
    assert ok(words, rows=4096, table=8192) == "" and ok(words, o=0, q=40000) == ""


def test_merge_and_logits_overlaps_by_place(host):
    merge = dict(part=8192, o=4096, os=512, n_head=4, n_shared=1, n_own=2, rows=20000, ts=4, n_seq=3, log2=5)
    ok = lambda bound, **k: _refuse(host, "attention_paged_merge", [128], list((merge | k).values()), bound)  # noqa: E731
    assert ok([ARENA, ARENA]) == "" and ok([ARENA, WORDS], rows=4096) == ""
    assert "overlap" in ok([ARENA, ARENA], rows=4096) and "control words" in ok([ARENA, ARENA], o=4)
    ok = lambda bound, **k: _refuse(host, "logits_adjust", [], _logits(**k), bound)  # noqa: E731
    assert ok([ARENA, ARENA]) == "" and ok([ARENA, WORDS], ctrl=8192, hist=8192, bias=8192, mask=8192) == ""
    for name in ("ctrl", "hist", "bias", "mask"):
        assert "overlap" in ok([ARENA, ARENA], **{name: 8192})
        assert "overlap" in ok([ARENA, (ARENA[0] + 4096, A)], **{name: 8192 - 1024})
    assert "control words" in ok([ARENA, ARENA], x=8192, y=0)
