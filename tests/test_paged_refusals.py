"""What csdr_paged_* and csdr_token_logprobs refuse, without a GPU: every refusal comes before a
launch, with a status and a message. And the page lookups of csrc/paged.hpp, compiled for the
host."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from conftest import ROOT
from cortexsdr_amd import _lib

INVALID, WORKSPACE, UNSUPPORTED = -1, -5, -6
P = 4096  # an aligned address that no refused call reads
OUT = 2 * P


def kv(**over):
    d = dict(k_pages=P, v_pages=P, page_table=P, lens=P, kv_dtype=1, page_size=16, n_pages=4,
             n_kv_heads=2, head_dim=64, n_seqs=2, table_stride=3)
    d.update(over)
    return C.byref(_lib.PagedKV(**d))


def refused(rc, status):
    assert rc == status
    assert _lib.load().csdr_last_error()


BAD_CACHE = [
    (dict(k_pages=None), INVALID), (dict(v_pages=None), INVALID),
    (dict(page_table=None), INVALID), (dict(lens=None), INVALID),
    (dict(kv_dtype=0), UNSUPPORTED), (dict(kv_dtype=3), UNSUPPORTED),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
    (dict(page_size=8), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
    (dict(page_size=8192), UNSUPPORTED), (dict(page_size=-16), UNSUPPORTED),
    (dict(n_pages=0), INVALID), (dict(n_kv_heads=0), INVALID), (dict(n_seqs=0), INVALID),
    (dict(n_seqs=-1), INVALID), (dict(table_stride=0), INVALID),
    (dict(table_stride=1 << 27), INVALID), (dict(k_pages=P + 8), INVALID),
]


@pytest.mark.parametrize("over,status", BAD_CACHE)
def test_bad_cache(over, status):
    lib = _lib.load()
    refused(lib.csdr_paged_append(kv(**over), P, P, P, 0, 2, None, 0, 4, 0, 0, 0, 1e4, P, None),
            status)
    refused(lib.csdr_paged_read(kv(**over), 2, None, 0, P, P, 0, None), status)
    refused(lib.csdr_paged_attn(kv(**over), P, 0, 2, None, 0, 4, 0, 0, 0.0, None, OUT, P, 1 << 40,
                                None), status)
    assert lib.csdr_paged_attn_workspace_bytes(kv(**over), 2, None, 0, 4, 0) == 0


def test_no_cache():
    lib = _lib.load()
    refused(lib.csdr_paged_read(None, 2, None, 0, P, P, 0, None), INVALID)


@pytest.mark.parametrize("n,starts,mq", [(0, None, 0), (-2, None, 0), (3, None, 0), (3, P, 0),
                                         (3, P, -1)])
def test_bad_tokens(n, starts, mq):
    lib = _lib.load()
    refused(lib.csdr_paged_append(kv(), P, P, P, 0, n, starts, mq, 4, 0, 0, 0, 1e4, P, None),
            INVALID)
    refused(lib.csdr_paged_read(kv(), n, starts, mq, P, P, 0, None), INVALID)
    refused(lib.csdr_paged_attn(kv(), P, 0, n, starts, mq, 4, 0, 0, 0.0, None, OUT, P, 1 << 40,
                                None), INVALID)


@pytest.mark.parametrize("over", [
    dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(dtype=2), dict(Hq=3),
    dict(Hq=0), dict(theta=-1.0), dict(theta=float("nan")), dict(theta=float("inf")),
    dict(qs=255), dict(ks=127), dict(vs=-128), dict(q_out=P, qs=512),
])
def test_bad_append(over):
    a = dict(q=P, k=P, v=P, dtype=0, Hq=4, qs=0, ks=0, vs=0, theta=1e4, q_out=OUT)
    a.update(over)
    refused(_lib.load().csdr_paged_append(kv(), a["q"], a["k"], a["v"], a["dtype"], 2, None, 0,
                                          a["Hq"], a["qs"], a["ks"], a["vs"], a["theta"],
                                          a["q_out"], None), INVALID)


@pytest.mark.parametrize("over", [
    dict(q=None), dict(out=None), dict(dtype=2), dict(Hq=3), dict(Hq=-4), dict(qs=255),
    dict(max_len=-1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(opt=_lib.AttnOptions(softcap=-1.0)), dict(opt=_lib.AttnOptions(softcap=float("inf"))),
    dict(opt=_lib.AttnOptions(softcap=float("nan"))), dict(opt=_lib.AttnOptions(window=-1)),
    dict(opt=_lib.AttnOptions(softcap=1e-40)), dict(out=P),
])
def test_bad_attn(over):
    a = dict(q=P, out=OUT, dtype=0, Hq=4, qs=0, max_len=0, scale=0.0, opt=None)
    a.update(over)
    opt = C.byref(a["opt"]) if a["opt"] is not None else None
    refused(_lib.load().csdr_paged_attn(kv(), a["q"], a["dtype"], 2, None, 0, a["Hq"], a["qs"],
                                        a["max_len"], a["scale"], opt, a["out"], P, 1 << 40,
                                        None), INVALID)


def test_too_many_tokens():
    """More workgroups than one launch may have."""
    lib = _lib.load()
    n, big = 1 << 27, kv(n_seqs=1 << 20)
    refused(lib.csdr_paged_append(big, P, P, P, 0, n, P, n, 4, 0, 0, 0, 1e4, OUT, None), INVALID)
    refused(lib.csdr_paged_read(big, n, P, n, P, OUT, 0, None), INVALID)
    # prompts; steps, joined by one workgroup per token and head
    refused(lib.csdr_paged_attn(big, P, 0, n, P, n, 4, 0, 0, 0.0, None, OUT, P, 1 << 60, None),
            INVALID)
    refused(lib.csdr_paged_attn(big, P, 0, n, P, 32, 4, 0, 0, 0.0, None, OUT, P, 1 << 60, None),
            INVALID)


def test_bad_read():
    lib = _lib.load()
    refused(lib.csdr_paged_read(kv(), 2, None, 0, None, P, 0, None), INVALID)
    refused(lib.csdr_paged_read(kv(), 2, None, 0, P, P, 2, None), INVALID)


def test_page_bytes():
    f = _lib.load().csdr_paged_page_bytes
    assert f(1, 16, 2, 64) == 16 * 2 * 64 * 2
    assert f(2, 64, 8, 128) == 64 * 8 * 128 * 5 // 8
    for bad in ((0, 16, 2, 64), (1, 8, 2, 64), (1, 48, 2, 64), (1, 16, 0, 64), (1, 16, 2, 80)):
        assert f(*bad) == 0


@pytest.mark.parametrize("over,status", [
    (dict(x=None), INVALID), (dict(rows=0), INVALID), (dict(n=0), INVALID),
    (dict(dtype=2), INVALID), (dict(top=-1), UNSUPPORTED), (dict(top=65), UNSUPPORTED),
    (dict(tokens=None), INVALID), (dict(lp=None), INVALID), (dict(ids=None), INVALID),
    (dict(tl=None), INVALID), (dict(stride=99), INVALID), (dict(t=float("nan")), INVALID),
    (dict(t=float("inf")), INVALID), (dict(t=1e-40), INVALID), (dict(rows=1 << 24), INVALID),
])
def test_bad_logprobs(over, status):
    a = dict(x=P, dtype=0, rows=2, n=100, stride=0, t=1.0, tokens=P, lp=P, h=P, top=3, ids=P, tl=P)
    a.update(over)
    refused(_lib.load().csdr_token_logprobs(
        a["x"], a["dtype"], a["rows"], a["n"], a["stride"], a["t"], a["tokens"], a["lp"], a["h"],
        a["top"], a["ids"], a["tl"], P, 1 << 40, None), status)


LOOKUPS = r"""
#include <cassert>
#include <climits>
#include "paged.hpp"
using namespace csdr;
int main() {
    const int32_t table[2 * 3] = {4, 0, -1, 5, INT_MIN, INT_MAX};
    int32_t lens[2] = {40, INT_MAX};
    int32_t start[3] = {0, 7, 9};
    PagedView pv{};
    pv.table = table;
    pv.lens = lens;
    pv.n_pages = 5;
    pv.shift = 4;
    pv.hkv = 2;
    pv.stride = 3;
    pv.n_seqs = 2;
    pv.n_tokens = 9;
    pv.max_q = 4;
    // ids outside [0, n_pages), positions outside the row
    assert(page_of(pv, 0, 0) == 4 && page_of(pv, 0, 31) == 0 && page_of(pv, 0, 32) == -1);
    assert(page_of(pv, 0, 48) == -1 && page_of(pv, 0, -1) == -1 && page_of(pv, 0, INT_MAX) == -1);
    assert(page_of(pv, 1, 0) == -1 && page_of(pv, 1, 16) == -1 && page_of(pv, 1, 32) == -1);
    // rows of a sequence: clamped to the call's tokens and to max_q
    pv.q_start = start;
    SeqRows r = seq_rows(pv, 0);
    assert(r.first == 0 && r.n == 4 && r.p0 == 33 && r.len == 40);
    r = seq_rows(pv, 1);
    assert(r.first == 7 && r.n == 2 && r.len <= kMaxPositions * 3LL / 2 && r.p0 == r.len - 2);
    const int bad[][3] = {{-3, INT_MAX, 5}, {8, 2, -1}, {INT_MIN, INT_MIN, INT_MAX}, {100, 3, 100}};
    for (auto& s : bad) {
        for (int i = 0; i < 3; ++i) start[i] = s[i];
        for (int b = 0; b < 2; ++b) {
            r = seq_rows(pv, b);
            assert(r.first >= 0 && r.n >= 0 && r.n <= pv.max_q && r.first + r.n <= pv.n_tokens);
        }
    }
    lens[0] = INT_MIN;
    r = seq_rows(pv, 0);
    assert(r.len == 0 && r.p0 <= 0);
    // every value of a head lies inside it, no two share bits
    for (int q4 = 0; q4 < 2; ++q4)
        for (int ps = 16; ps <= 64; ps *= 2) {
            const int n = paged_head_bytes(q4, ps, 128);
            static bool used[2][128 * 64 * 8];
            for (auto& u : used)
                for (bool& x : u) x = false;
            for (int slot = 0; slot < ps; ++slot)
                for (int d = 0; d < 128; ++d) {
                    if (!q4) continue;
                    const int kb = 32 * k_word<128>(slot, d & ~7) + code_shift(d & 7);
                    const int vb = 32 * v_word<128>(slot, d) + code_shift(slot & 7);
                    assert(kb + 4 <= 8 * scale_offset(128, ps, 0, 0) && !used[0][kb / 4]);
                    assert(vb + 4 <= 8 * scale_offset(128, ps, 0, 0) && !used[1][vb / 4]);
                    used[0][kb / 4] = used[1][vb / 4] = true;
                    assert(min_offset(128, ps, d / 32, slot) + 2 <= n);
                }
            if (q4) assert(min_offset(128, ps, 3, ps - 1) + 2 == n);
        }
    return 0;
}
"""


def test_lookups_on_the_host(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src = tmp_path / "lookups.cpp"
    src.write_text(LOOKUPS)
    exe = tmp_path / "lookups"
    r = subprocess.run([hipcc, "-std=c++17", "-O1", "--offload-arch=gfx950", "-x", "hip",
                        "-I" + os.path.join(ROOT, "cortexsdr_amd", "csrc"), str(src), "-o",
                        str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
