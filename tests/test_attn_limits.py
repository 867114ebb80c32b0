"""Limits of attention's sizes on the host: bounds of nought, and lengths next to 2^31."""
import ctypes
import os
import subprocess

import pytest

from nebula_b200 import _lib
from test_attn_api import ROOT, shape


def size(sh, max_kv, prefix=0):
    return _lib.lib().hq_attn_paged_workspace_size(ctypes.byref(sh), max_kv, prefix)


@pytest.mark.parametrize("heads", [(40, 8), (64, 1), (17, 1), (128, 1)])
@pytest.mark.parametrize("seqs", [1, 3])
def test_a_bound_of_no_rows_plans_as_one_of_one(heads, seqs):
    """A sequence may have more rows than max_q_len, and is reported or computed: a call with a bound of 0 launches what
    one with 1 does, with its workspace."""
    kw = dict(n_tokens=seqs, n_seqs=seqs, n_heads=heads[0], n_kv_heads=heads[1], head_dim=128)
    for max_kv in (100, 20000):
        assert size(shape(max_q_len=0, **kw), max_kv) == size(shape(max_q_len=1, **kw), max_kv)
    assert size(shape(max_q_len=0, **kw), 20000) > 0


@pytest.mark.parametrize("heads,rows", [((40, 8), 1), ((10, 2), 30), ((64, 1), 1), ((8, 8), 4)])
def test_a_bound_of_keys_next_to_the_largest(heads, rows):
    """max_kv_len is often the longest there can be: it plans as one of a few keys less."""
    for seqs in (1, 70):
        sh = shape(n_tokens=seqs * rows, n_seqs=seqs, max_q_len=rows, n_heads=heads[0], n_kv_heads=heads[1], head_dim=128)
        want = size(sh, 2 ** 31 - 1000)
        assert want > 0
        for bound in (2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 16, 2 ** 31 - 1):
            assert size(sh, bound) == want


def test_tiles_of_the_longest_sequences(tmp_path):
    """Tiles and boxes of keys next to 2^31, in the functions that the kernels use, compiled for the host."""
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include "hq_attn_index.h"
#include <cstdio>
#include <climits>
#include <initializer_list>
using namespace hq;
#define CHECK(x) do { if (!(x)) { std::printf("%d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    for (int unit : {16, 32, 64, 128, 256})
        for (long long keys : {0LL, 1LL, 2LL, 15LL, 16LL, 17LL, 127LL, 128LL, 129LL, 1000LL, (long long)INT_MAX, INT_MAX - 1LL,
                               INT_MAX - 15LL, INT_MAX - 63LL, INT_MAX - 126LL, INT_MAX - 127LL, INT_MAX - 128LL})
            CHECK(key_tiles((int)keys, unit) == (keys + unit - 1) / unit);
    CHECK(sees_any(0, 0) == false && sees_any(1, 0) && sees_any(0, 1) && sees_any(INT_MAX, INT_MAX) && sees_any(5, INT_MAX));
    return 0;
}''')
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "nebula_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
