"""CPU tests of the launches that the batch operators' dispatches become (runtime/batch.h): every
head, row, part and token has its workgroup, and each form is taken on its side of its line."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from skyla_hip import batch as B
from test_host_batch import RUNTIME, _append, _attend, _logits
from test_host_batch_words import u32

SHIM = r"""
#include "batch.h"
extern "C" int shape(const char *name, const uint32_t *spec, const uint32_t *w, uint32_t rows, uint32_t *out) {
  const batch::Shape s = batch::shape(batch::op_of(name), spec, w, rows);
  std::copy(s.groups, s.groups + 3, out);
  out[3] = s.threads;
  out[4] = s.form;
  out[5] = (uint32_t)s.extra.size();
  std::copy(s.extra.begin(), s.extra.end(), out + 6);
  return 0;
}
extern "C" int other(const char *name, const char *symbol, char *to) {
  const std::string s = batch::other_form(batch::op_of(name), symbol);
  std::strcpy(to, s.c_str());
  return 0;
}
"""


@pytest.fixture(scope="module")
def shape(tmp_path_factory):
    d = tmp_path_factory.mktemp("launch")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", RUNTIME, "-o", str(so),
                    str(src)], check=True)
    lib = C.CDLL(str(so))

    def run(name, spec, words, rows):
        out = (C.c_uint32 * 8)()
        lib.shape(name.encode(), u32(spec), u32(words), rows, out)
        return list(out[:3]), out[3], out[4], list(out[6:6 + out[5]])
    run.lib = lib
    return run


def test_the_other_forms_names(shape):
    to = C.create_string_buffer(64)
    for name, symbol, want in (("kv_append", "kv_append__0_1_128", "kv_append_4__0_1_128"),
                               ("kv_append", "kv_append__1_1_128", "kv_append_4__1_1_128"),
                               ("attention_paged", "attention_paged__4_0_1_128", "attention_paged__4_0_1_128"),
                               ("attention_paged_merge", "attention_paged_merge__128", "attention_paged_merge_8__128"),
                               ("logits_adjust", "logits_adjust_256", "logits_adjust_1024")):
        shape.lib.other(name.encode(), symbol.encode(), to)
        assert to.value.decode() == want


@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (4, 2), (16, 8), (32, 8), (32, 4), (12, 3), (1024, 1024)])
def test_append(shape, n_head, n_kv):
    heads = n_head + 2 * n_kv
    for rows in (1, 7, 128, 341, 342, 1365, 1366, 2048, 65535):
        g, threads, form, extra = shape("kv_append", [0, 1, 128], _append(n_head=n_head, n_kv=n_kv), rows)
        assert g[1:] == [rows, 1] and threads == 256 and extra == []
        assert form == (rows * -(-heads // 16) >= 4096)
        per = 64 if form else 16
        assert g[0] * per >= heads > (g[0] - 1) * per  # no head without a workgroup, no workgroup without a head


@pytest.mark.parametrize("n_kv,rep", [(1, 1), (8, 4), (4, 8), (3, 2), (8, 1)])
@pytest.mark.parametrize("n_shared,n_own", [(0, 1), (1, 1), (5, 3), (8, 2), (33, 1), (100, 128)])
def test_attention(shape, n_kv, rep, n_shared, n_own):
    for rows in (1, 2, 15, 17, 31, 33, 127, 128, 129):
        for wide in (0, 1):
            words = _attend(n_kv=n_kv, n_shared=n_shared, n_own=n_own, wide=wide)
            g, threads, form, extra = shape("attention_paged", [rep, 0, 1, 128], words, rows)
            assert g[1:] == [1, 1] and threads == 256 and form == 0 and extra == [rows]
            tile = 128 if wide and n_shared else 16
            tiles, groups, own = -(-rows * rep // tile), n_kv * n_shared, rows * n_kv * n_own
            if tile == 16:
                assert g[0] == groups * tiles + own
                continue
            # the kernel's map: the tiles of a (part, key head) 8 workgroups apart, each once
            first = -(-groups // 8) * 8 * tiles
            assert g[0] == first + own
            w = np.arange(first)
            at, t = w // (8 * tiles) * 8 + w % 8, w // 8 % tiles
            seen = np.bincount((at * tiles + t)[at < groups], minlength=groups * tiles)
            assert seen.size == groups * tiles and (seen == 1).all()


def test_merge(shape):
    for n_head in (1, 4, 16, 30, 32, 512, 513, 8192):
        for rows in (1, 2, 16, 17, 128):
            for n_shared, n_own in ((0, 2), (15, 1), (16, 1), (8, 9), (512, 512)):
                words = [8192, 4096, 512, n_head, n_shared, n_own, 20000, 4, 3, 5]
                g, threads, form, extra = shape("attention_paged_merge", [128], words, rows)
                assert form == (n_shared + n_own > 16 and rows * n_head <= 512) and extra == []
                assert threads == (512 if form else 256) and g == [n_head if form else -(-n_head // 4), rows, 1]


@pytest.mark.parametrize("v", [1, 1000, 4096, 4097, 16384, 16385, 151936])
def test_logits(shape, v):
    for rows in (1, 48, 128):
        for stride in (0, 8188, 8192, 32768):
            g, threads, form, extra = shape("logits_adjust", [0], _logits(v=v, hs=stride), rows)
            assert form == (stride >= 8192) and threads == (1024 if form else 256) and extra == []
            assert g == [-(-v // (16 * threads)), rows, 1]


def test_the_shared_runs_form():
    """128 query rows a workgroup on their side of the line, by key heads, query rows and positions."""
    for n_kv, rep, rows, shared, wide in ((8, 4, 16, 2000, False), (8, 4, 16, 4000, True), (8, 4, 32, 1000, False),
                                          (8, 4, 32, 2000, True), (4, 8, 32, 1000, False), (2, 8, 64, 2000, True),
                                          (2, 8, 64, 1000, False), (8, 2, 16, 100000, False), (8, 1, 64, 3500, True),
                                          (1, 1, 64, 24575, False), (1, 1, 64, 24576, True)):
        assert B.splits(rows, n_kv, rep, shared, 1).wide == wide, (n_kv, rep, rows, shared)
