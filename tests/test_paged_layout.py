"""The layout of a page (cortexsdr_hip.h): offsets on the host for every shape, and the bytes that
an append leaves, read one by one."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from conftest import ROOT

LAYOUT = r"""
#include <cassert>
#include <vector>
#include "paged.hpp"
using namespace csdr;
// every byte (4 bits: half byte) of a head belongs to one value, scale or minimum, and none is left
template <int HD>
void check(int ps) {
    const int bytes = paged_head_bytes(true, ps, HD);
    std::vector<char> k(2 * bytes), v(2 * bytes);
    auto use = [&](std::vector<char>& u, int from, int n) {
        for (int i = from; i < from + n; ++i) {
            assert(i >= 0 && i < 2 * bytes && !u[i]);
            u[i] = 1;
        }
    };
    for (int slot = 0; slot < ps; ++slot) {
        for (int d = 0; d < HD; ++d) {
            use(k, 8 * k_word<HD>(slot, d & ~7) + code_shift(d & 7) / 4, 1);
            use(v, 8 * v_word<HD>(slot, d) + code_shift(slot & 7) / 4, 1);
        }
        for (int g = 0; g < HD / kGroup; ++g)
            for (auto* u : {&k, &v}) {
                use(*u, 2 * scale_offset(HD, ps, g, slot), 4);
                use(*u, 2 * min_offset(HD, ps, g, slot), 4);
            }
    }
    for (int i = 0; i < 2 * bytes; ++i) assert(k[i] && v[i]);
    assert(bytes % 16 == 0 && paged_head_bytes(false, ps, HD) == ps * HD * 2);
}
int main() {
    for (int ps = 16; ps <= 4096; ps *= 2) {
        check<64>(ps);
        check<128>(ps);
    }
    return 0;
}
"""


def test_every_byte_of_a_page_once(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, exe = tmp_path / "layout.cpp", tmp_path / "layout"
    src.write_text(LAYOUT)
    r = subprocess.run([hipcc, "-std=c++17", "-O1", "--offload-arch=gfx950", "-x", "hip",
                        "-I" + os.path.join(ROOT, "cortexsdr_amd", "csrc"), str(src), "-o",
                        str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ps", [16, 128])
def test_bytes_of_an_append(gpu, kv, hd, ps):
    """Each value where the header puts it."""
    from test_paged_gpu import Setup

    s = Setup(gpu, [150], (2, 2, hd), kv, ps=ps, seed=71)
    s.append([141], with_q=False)
    table = s.table.cpu().numpy()[0]
    for pool, held, is_v in ((s.cache.k, s.k[0], False), (s.cache.v, s.v[0], True)):
        pages = pool.cpu().numpy().reshape(s.cache.n_pages, 2, -1)
        for p in range(141):
            t = p % ps
            for h in range(2):
                head = np.ascontiguousarray(pages[table[p // ps], h])
                f, d = head.view(np.float16), np.arange(hd)
                if kv == "f16":
                    got = f[(t // 8 * hd + d) * 8 + t % 8] if is_v else f[t * hd + d]
                else:
                    w = t // 8 * hd + d % 16 * (hd // 16) + d // 16 if is_v else \
                        t * (hd // 8) + d % 32 // 8 * (hd // 32) + d // 32
                    e = np.full(hd, t % 8) if is_v else d % 8
                    code = head.view(np.uint32)[w] >> (4 * (e // 2) + 16 * (e % 2)).astype(np.uint32)
                    par = ps * hd // 4 + d // 32 * ps + t
                    got = f[par + ps * (hd // 32)].astype(np.float32) + \
                        f[par].astype(np.float32) * (code & 15).astype(np.float32)
                assert np.array_equal(got.astype(np.float32), held[p, h])
