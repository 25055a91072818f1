"""Which sets of rows share memory: the host's arithmetic against brute force, and the refusals that go by it.  No GPU."""
from __future__ import annotations

import ctypes
import subprocess

import pytest
from conftest import PKG
from test_paged_cpu import view

PROGRAM = r'''
#include "q3_rows_meet.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace q3;
static bool share(const RowSet& a, const RowSet& b, bool same) {
    for (int i = 0; i < a.tokens; ++i) for (int k = 0; k < a.heads; ++k)
        for (int j = 0; j < b.tokens; ++j) for (int l = 0; l < b.heads; ++l) {
            if (same && i == j && k == l) continue;
            const long long x = (long long)a.address + i * a.token_stride + k * a.head_stride, y = (long long)b.address + j * b.token_stride + l * b.head_stride;
            if (x < y + b.width && y < x + a.width) return true;
        }
    return false;
}
int main() {
    srand(1);
    long yes = 0, no = 0, unknown = 0, self = 0;
    for (int it = 0; it < 200000; ++it) {
        auto pick = [](int n) { return rand() % n; };
        RowSet a, b;
        a.tokens = 1 + pick(5); b.tokens = 1 + pick(5); a.heads = 1 + pick(4); b.heads = pick(2) ? a.heads : 1 + pick(4);
        a.width = 8 << pick(2); b.width = 8 << pick(2);
        a.token_stride = 4 * pick(24); a.head_stride = 4 * pick(24);
        b.token_stride = pick(4) ? a.token_stride : 4 * pick(24); b.head_stride = pick(3) ? a.head_stride : 4 * pick(24);
        a.address = 1000; b.address = 1000 + 4 * (pick(160) - 80);
        const bool truth = share(a, b, false);
        const Meet m = rows_meet(a, b), n = rows_meet(b, a);
        if (m != n) { puts("not symmetric"); return 1; }
        if (m == Meet::Unknown) { ++unknown; if (a.token_stride == b.token_stride || a.tokens == 1 || b.tokens == 1) { puts("unknown"); return 1; } }
        else if ((m == Meet::Yes) != truth) { printf("%d %d: %d\n", (int)m, (int)truth, it); return 1; }
        else ++(truth ? yes : no);
        const bool s = share(a, a, true);
        if (rows_meet_themselves(a) != s) { printf("themselves %d\n", it); return 1; }
        self += s;
    }
    // sizes whose products leave 64 bits
    RowSet big{1ull << 40, 1ll << 40, 1ll << 40, 0x7fffffff, 1024, 256}, one{(1ull << 40) + (1ull << 50), 0, 0, 1, 1, 256}, off{(1ull << 40) + (1ull << 50) + 256, 0, 0, 1, 1, 256};
    if (rows_meet(big, one) != Meet::Yes || rows_meet(big, off) != Meet::No || !rows_meet_themselves(big)) { puts("large"); return 1; }
    if (yes < 1000 || no < 1000 || unknown < 1000 || self < 1000) { puts("nothing tested"); return 1; }
    puts("ok");
}
'''


def test_against_brute_force(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{PKG / 'csrc'}", "-o", str(tmp_path / "t"), str(tmp_path / "t.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "t")], capture_output=True, text=True).stdout.strip() == "ok"


ATTN = dict(q=1 << 24, out=1 << 26, q_token=2048, q_head=128, out_token=2048, out_head=128, q_heads=16, scale=0.1, workspace=1 << 28, workspace_bytes=0)


@pytest.mark.parametrize("change", [dict(out=(1 << 24) + 256), dict(out=(1 << 24) + 4096), dict(out=(1 << 24) - 4096 + 16), dict(out=(1 << 24) + 4096 * 2 + 15 * 256), dict(out_token=128),
                                    dict(q_token=4096, out=(1 << 24) + 4096 + 15 * 256, out_token=4096), dict(out=(1 << 24) + 4096, out_token=4096), dict(out_token=1024, out_head=512)])
def test_attention_refuses_rows_that_overlap(change):
    from qwen3mk import _cabi

    lib = _cabi.load()
    rc = lib.q3_paged_attn(ctypes.byref(view()), ctypes.byref(_cabi.PagedAttnArgs(**{**ATTN, **change})), None)
    assert rc == _cabi.ERR_INVALID and b"overlap" in lib.q3_last_error(None)


@pytest.mark.parametrize("change", [{}, dict(out=(1 << 24) + 3 * 4096), dict(q_token=4096, out=(1 << 24) + 4096, out_token=4096), dict(q_head=256, q_token=8192, out=(1 << 24) + 256, out_head=256, out_token=8192),
                                    dict(out_token=128, out_head=3 * 128)])
def test_attention_takes_rows_that_lie_beside_one_another(change):
    """As far as the workspace, which is asked for last: no GPU is here to run on."""
    from qwen3mk import _cabi

    lib = _cabi.load()
    lib.q3_paged_attn(ctypes.byref(view()), ctypes.byref(_cabi.PagedAttnArgs(**{**ATTN, **change})), None)
    assert b"workspace" in lib.q3_last_error(None)


ROPE = dict(q=1 << 24, k=(1 << 24) + 16 * 256, v=(1 << 24) + 24 * 256, q_out=1 << 26, q_token=4096, q_head=128, k_token=4096, k_head=128, v_token=4096, v_head=128, out_token=2048, out_head=128,
            q_heads=16, rows_type=0, rope_positions=0, rotary_dim=0, eps=-1.0)      # the last one is refused behind the overlaps' turn: nothing is launched where a GPU is
IN_PLACE = dict(q_out=1 << 24, out_token=4096)


@pytest.mark.parametrize("change", [dict(q_out=1 << 24), dict(q_out=(1 << 24) + 256, out_token=4096), dict(q_out=(1 << 24) + 16 * 256, out_token=4096), dict(q_out=(1 << 24) + 24 * 256 - 8, out_token=4096),
                                    {**IN_PLACE, "rows_type": 1}, {**IN_PLACE, "rows_type": 2}, {**IN_PLACE, "q_head": 256, "q_token": 8192}, dict(out_token=256)])
def test_rope_refuses_rows_that_overlap(change):
    from qwen3mk import _cabi

    lib = _cabi.load()
    assert lib.q3_paged_rope(ctypes.byref(view()), ctypes.byref(_cabi.PagedRopeArgs(**{**ROPE, **change})), None) == _cabi.ERR_INVALID
    assert b"overlap" in lib.q3_last_error(None)


@pytest.mark.parametrize("change", [{}, IN_PLACE, dict(q_out=(1 << 24) - 3 * 8192), dict(q_out=(1 << 24) + 3 * 8192), dict(q_token=8192, k_token=8192, v_token=8192, q_out=(1 << 24) + 8192, out_token=8192),
                                    {**IN_PLACE, "k": None, "v": None}, dict(q_out=(1 << 24) + 8192, q_token=0, out_token=4096)])      # (the last: one row of q for all tokens)
def test_rope_takes_rows_that_lie_beside_one_another(change):
    from qwen3mk import _cabi

    lib = _cabi.load()
    assert lib.q3_paged_rope(ctypes.byref(view()), ctypes.byref(_cabi.PagedRopeArgs(**{**ROPE, **change})), None) == _cabi.ERR_INVALID
    assert b"eps" in lib.q3_last_error(None)
