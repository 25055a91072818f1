"""The paged operators' host side: how work is dealt out (brute force on the CPU), rotary tables, refusals of the C ABI.  No GPU."""
from __future__ import annotations

import ctypes
import math
import subprocess

import pytest
import torch

from conftest import PKG

PLAN = r'''
#include "q3_paged_plan.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace q3;
static int fail(const char* what) { puts(what); return 1; }
int main() {
    srand(1);
    for (int it = 0; it < 20000; ++it) {
        PgShape s;
        const int log = 6 + rand() % 2;
        s.unit_log = log; s.tile_log = rand() % (log + 1); s.heads = 1 + rand() % 8; s.batch = 1 + rand() % 6;
        std::vector<int> qs(s.batch + 1), kv(s.batch);
        qs[0] = rand() % 4 ? 0 : rand() % 9;
        for (int b = 0; b < s.batch; ++b) {
            const int q = rand() % 3 == 0 ? 0 : rand() % (rand() % 2 ? 5 : 400);
            qs[b + 1] = qs[b] + q;
            kv[b] = rand() % 4 ? q + rand() % 1000 : rand() % (q + 1);
        }
        s.n_tokens = qs[s.batch] - (rand() % 5 == 0 ? rand() % 7 : 0);
        if (s.n_tokens < 0) s.n_tokens = 0;
        s.most_keys = rand() % 5 ? 100000 : rand() % 900;
        if (rand() % 10 == 0) kv[rand() % s.batch] = rand() % 2 ? -5 : 2147483647;      // descriptors that say nonsense
        if (rand() % 10 == 0) qs[rand() % (s.batch + 1)] = rand() % 2 ? -2147483647 : 2147483647;
        std::vector<long long> p(s.batch + 1);
        std::vector<PgSegment> items;
        std::vector<int> owner(s.n_tokens + 1, 0);
        for (int b = 0; b < s.batch; ++b) {
            const PgSeq q = pg_seq(s, qs.data(), kv.data(), b);
            if (q.q0 < 0 || q.q < 0 || q.q0 + q.q > s.n_tokens || q.kv < 0 || q.kv > s.most_keys) return fail("descriptors");
            long long u = 0;
            for (int r = 0; r < pg_tiles(s, q); ++r) {
                if (pg_units_before(s, q, r) != u) return fail("units before a tile");
                if ((pg_tile_units(s, q, r) << s.unit_log) < q.kv - q.q + (r + 1 < pg_tiles(s, q) ? (r + 1) << s.tile_log : q.q)) return fail("a tile sees keys that no unit holds");
                u += pg_tile_units(s, q, r);
            }
            if (u != pg_head_units(s, q)) return fail("units of a head");
            p[b + 1] = p[b] + u * s.heads;
            for (int h = 0; h < s.heads; ++h)
                for (int r = 0; r < pg_tiles(s, q); ++r) {
                    PgSegment g{};
                    g.b = b; g.h = h; g.r = r; g.units = (int)pg_tile_units(s, q, r);
                    items.push_back(g);
                }
        }
        const long long total = p[s.batch];
        if (!total) continue;
        const int n = pg_blocks(total, 1 + rand() % 300, 1 + rand() % 3);
        size_t at = 0;
        int k = 0;
        for (int i = 0; i < n; ++i) {
            PgWalk w;
            int cut = 0, segment = 0;
            if (w.begin(s, p.data(), qs.data(), kv.data(), pg_run_start(total, n, i), pg_run_start(total, n, i + 1))) do {
                if (at >= items.size()) return fail("more segments than items");
                const PgSegment &g = items[at], &x = w.s;
                if (g.b != x.b || g.h != x.h || g.r != x.r || x.k0 != k || x.units != g.units || x.k1 <= x.k0 || x.k1 > x.units) return fail("segment");
                k = x.k1;
                if (k == g.units) { k = 0; ++at; }
                if (!w.whole()) ++cut;
                int runs = 0;
                while (runs < n && pg_run_start(total, n, runs) < w.at + x.units - x.k0) ++runs;
                if (pg_runs_before(total, n, w.at + x.units - x.k0) != runs) return fail("runs before the end of an item");
                ++segment;
            } while (w.next(s, qs.data(), kv.data()));
            if (cut > 2 || !segment) return fail("a run holds more than two parts of items, or nothing");
        }
        if (at != items.size() || k) return fail("items are left");
    }
    puts("ok");
}
'''


def test_every_unit_is_dealt_out_once(tmp_path):
    src = tmp_path / "plan.cpp"
    src.write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", str(PKG / "csrc"), str(src), "-o", str(tmp_path / "plan")], check=True)
    got = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True)
    assert got.stdout.strip() == "ok" and got.returncode == 0, got.stdout + got.stderr


def test_rope_table_without_scaling_is_the_engines():
    from qwen3mk import kernel, paged

    assert torch.equal(paged.rope_table(300, "cpu"), kernel.rope_rows(300, "cpu"))
    half = paged.rope_table(50, "cpu", rotary_dim=32, theta=1e4)
    assert half.shape == (50, 32)
    assert float(half[49, 3]) == pytest.approx(math.cos(49 * 1e4 ** (-6 / 32)), abs=2 ** -24) and float(half[49, 16 + 3]) == pytest.approx(math.sin(49 * 1e4 ** (-6 / 32)), abs=2 ** -24)


def test_rope_table_far_positions_keep_their_angles():
    """Position 131071: an angle of 1.3e5 in fp32 would be off by up to 2^-8; the table is off by its own rounding, 2^-25."""
    from qwen3mk import paged

    t = paged.rope_table(131072, "cpu", rotary_dim=4)
    assert float(t[131071, 0]) == pytest.approx(math.cos(131071.0), abs=2 ** -24) and float(t[131071, 2]) == pytest.approx(math.sin(131071.0), abs=2 ** -24)


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, {"type": "yarn", "factor": 4.0, "original": 32768},
                                     {"type": "llama3", "factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0}])
def test_scaled_frequencies(scaling):
    """Fastest and slowest frequencies, the ramp between them, and the factor on cosines and sines, from the definitions."""
    from qwen3mk import paged

    theta, r = 1e6, 128
    t = paged.rope_table(2, "cpu", scaling=scaling).double()
    gain = 0.1 * math.log(4.0) + 1 if scaling["type"] == "yarn" else 1.0
    assert torch.allclose(t[0, :64], torch.full((64,), gain, dtype=torch.float64), atol=1e-7) and not t[0, 64:].any()
    got = torch.atan2(t[1, 64:], t[1, :64])
    plain = torch.tensor([theta ** (-2 * i / r) for i in range(64)], dtype=torch.float64)
    ratio = got / plain
    factor = scaling["factor"]
    if scaling["type"] == "linear":
        assert torch.allclose(ratio, torch.full_like(ratio, 1 / factor), rtol=1e-6)
        return
    turns = scaling["original"] * plain / (2 * math.pi)
    fast, slow = (32, 1) if scaling["type"] == "yarn" else (4, 1)
    # (yarn's ramp begins and ends at whole indices: one further at most)
    inside = (turns < fast * 1.5) & (turns > slow / 1.5)
    assert torch.allclose(ratio[(turns > fast) & ~inside], torch.ones(1, dtype=torch.float64), rtol=1e-6)
    assert torch.allclose(ratio[(turns < slow) & ~inside], torch.full((1,), 1 / factor, dtype=torch.float64), rtol=1e-6)
    assert (ratio[1:] <= ratio[:-1] * (1 + 1e-6)).all() and 0.3 < float(ratio[inside].mean()) < 0.8


def test_ntk_keeps_the_fastest_and_divides_the_slowest():
    from qwen3mk import paged

    t = paged.rope_table(2, "cpu", scaling={"type": "ntk", "factor": 4.0}).double()
    got = torch.atan2(t[1, 64:], t[1, :64])
    assert float(got[0]) == pytest.approx(1.0, rel=1e-6) and float(got[63]) == pytest.approx(1e6 ** (-126 / 128) / 4, rel=1e-5)


def test_rope_table_refusals():
    from qwen3mk import paged

    for kw in ({"rotary_dim": 7}, {"rotary_dim": 0}, {"rotary_dim": 130}, {"scaling": {"type": "linear"}}, {"scaling": {"type": "linear", "factor": 0.5}},
               {"scaling": {"type": "yarn", "factor": 2.0}}, {"scaling": {"type": "other", "factor": 2.0}}, {"scaling": {"type": "linear", "factor": 2.0, "original": 5}}):
        with pytest.raises(ValueError):
            paged.rope_table(4, "cpu", **kw)
    with pytest.raises(ValueError):
        paged.rope_table(0, "cpu")


def test_pool_and_batch_refusals():
    from qwen3mk import paged

    k = torch.zeros(1, 4, 16, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.PagePool(k, k)
    for other in (k.half(), k[:, :2], torch.zeros(1, 4, 8, 16, 128, dtype=torch.bfloat16).transpose(2, 3)):
        with pytest.raises(ValueError, match="alike"):
            paged.PagePool(k, other)


def view(**kw):
    """A descriptor that passes every check (addresses that nothing reads), with changes."""
    from qwen3mk import _cabi

    base = dict(k_pages=1 << 20, v_pages=1 << 21, page_table=64, q_start=64, kv_len=64, page_stride=16 * 1024, slot_stride=1024, head_stride=128, table_stride=4, table_pages=4,
                n_pages=10, page_size=16, batch=2, n_tokens=3, max_new=2, kv_heads=8, type=0)
    return _cabi.Paged(**{**base, **kw})


BAD_VIEWS = [dict(k_pages=None), dict(v_pages=None), dict(page_table=None), dict(q_start=None), dict(kv_len=None), dict(page_size=24), dict(page_size=8), dict(page_size=512),
             dict(batch=0), dict(batch=1025), dict(n_pages=0), dict(table_pages=0), dict(table_stride=3), dict(n_tokens=-1), dict(max_new=-1), dict(kv_heads=0), dict(type=2),
             dict(k_pages=(1 << 20) + 2), dict(page_stride=16 * 1024 + 4), dict(slot_stride=-8), dict(head_stride=4), dict(page_table=65), dict(table_pages=1 << 28, table_stride=1 << 28)]


@pytest.mark.parametrize("bad", range(len(BAD_VIEWS)))
def test_bad_descriptors_are_refused(bad):
    from qwen3mk import _cabi

    lib = _cabi.load()
    c = view(**BAD_VIEWS[bad])
    attn = _cabi.PagedAttnArgs(q=1 << 20, out=1 << 20, q_token=2048, q_head=128, out_token=2048, out_head=128, q_heads=16, scale=0.1, workspace=1 << 20, workspace_bytes=1 << 40)
    rope = _cabi.PagedRopeArgs(q=1 << 20, k=1 << 20, v=1 << 20, q_out=1 << 20, q_heads=16, rows_type=2, rope_positions=5, rotary_dim=128, rope=1 << 20)
    assert lib.q3_paged_attn(ctypes.byref(c), ctypes.byref(attn), None) == _cabi.ERR_INVALID and lib.q3_last_error(None).startswith(b"q3_paged_attn: ")
    assert lib.q3_paged_rope(ctypes.byref(c), ctypes.byref(rope), None) == _cabi.ERR_INVALID and lib.q3_last_error(None).startswith(b"q3_paged_rope: ")


def test_bad_arguments_are_refused():
    from qwen3mk import _cabi

    lib, c = _cabi.load(), view()
    attn = dict(q=1 << 20, out=1 << 20, q_token=2048, q_head=128, out_token=2048, out_head=128, q_heads=16, scale=0.1, workspace=1 << 20, workspace_bytes=1 << 40)
    for bad in (dict(q=None), dict(out=None), dict(workspace=None), dict(q_heads=0), dict(q_heads=24), dict(q_heads=128), dict(q_heads=-16), dict(scale=0.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(q=(1 << 20) + 8), dict(q_token=2044), dict(out_head=-128)):
        assert lib.q3_paged_attn(ctypes.byref(c), ctypes.byref(_cabi.PagedAttnArgs(**{**attn, **bad})), None) == _cabi.ERR_INVALID, bad
    assert lib.q3_paged_attn(ctypes.byref(c), None, None) == _cabi.ERR_INVALID and lib.q3_paged_attn(None, None, None) == _cabi.ERR_INVALID
    rope = dict(q=1 << 20, k=1 << 20, v=1 << 20, q_out=1 << 20, q_token=4096, q_head=128, k_token=4096, k_head=128, v_token=4096, v_head=128, out_token=2048, out_head=128, q_heads=16,
                rows_type=2, rope_positions=5, rotary_dim=128, rope=1 << 20, eps=1e-6)
    for bad in (dict(q=None, k=None, v=None), dict(k=None), dict(q_out=None), dict(q_heads=0), dict(rows_type=3), dict(rotary_dim=12), dict(rotary_dim=136), dict(rotary_dim=-8), dict(rope=None),
                dict(rope_positions=0), dict(eps=-1.0), dict(eps=float("nan")), dict(q=(1 << 20) + 8), dict(rope=(1 << 20) + 2), dict(q_out=(1 << 20) + 4), dict(k_token=4098), dict(v_head=-4)):
        assert lib.q3_paged_rope(ctypes.byref(c), ctypes.byref(_cabi.PagedRopeArgs(**{**rope, **bad})), None) == _cabi.ERR_INVALID, bad
    assert lib.q3_paged_rope(ctypes.byref(c), None, None) == _cabi.ERR_INVALID and lib.q3_paged_rope(None, None, None) == _cabi.ERR_INVALID
    # no token: nothing to do, nothing is asked of the device
    none = view(n_tokens=0)
    assert lib.q3_paged_attn(ctypes.byref(none), ctypes.byref(_cabi.PagedAttnArgs(**attn)), None) == 0 and lib.q3_paged_rope(ctypes.byref(none), ctypes.byref(_cabi.PagedRopeArgs(**rope)), None) == 0


def test_struct_layouts():
    from qwen3mk import _cabi

    assert ctypes.sizeof(_cabi.Paged) == 5 * 8 + 4 * 8 + 8 * 4 and _cabi.Paged.type.offset == 100
    assert ctypes.sizeof(_cabi.PagedAttnArgs) == 2 * 8 + 4 * 8 + 8 + 3 * 8
    assert ctypes.sizeof(_cabi.PagedRopeArgs) == 4 * 8 + 8 * 8 + 4 * 8 + 6 * 4


def test_bad_limits_and_status_words_are_refused():
    from qwen3mk import _cabi

    lib, c = _cabi.load(), view()
    attn = dict(q=1 << 20, out=1 << 21, q_token=2048, q_head=128, out_token=2048, out_head=128, q_heads=16, scale=0.1, workspace=1 << 22, workspace_bytes=1 << 40)
    for limit, change in ((-1, {}), (5, dict(status=(1 << 20) + 2)), (5, dict(q=None))):
        assert lib.q3_paged_attn_limited(ctypes.byref(c), ctypes.byref(_cabi.PagedAttnArgs(**{**attn, **change})), limit, None) == _cabi.ERR_INVALID
        assert lib.q3_last_error(None).startswith(b"q3_paged_attn: ")
    assert lib.q3_paged_attn_limited(ctypes.byref(view(n_tokens=0)), ctypes.byref(_cabi.PagedAttnArgs(**attn)), 7, None) == 0
