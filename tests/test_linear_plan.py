"""How the linear operators cut their products (brimkern_b200/csrc/linear_plan.h), walked on the CPU: the
plan is host code, compiled here as it is."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "brimkern_b200", "csrc")
SMS = 148
# Clusters of 0 .. 8 CTAs that fit at once: more and fewer than a B200 takes, and none at all.
CLUSTERS = [(0, 148, 74, 48, 36, 28, 24, 20, 18), (0, 148, 74, 46, 32, 26, 20, 16, 14), (0, 148, 72, 0, 0, 0, 0, 0, 0)]
FIELDS = ("pair", "ranged", "drain", "cs", "nt_kernel", "nt", "f_rows", "half_cols", "tiles_m", "nk", "kb", "stages",
          "drain_steps", "ctas", "tiles", "tiles_whole", "range_units", "range_extra", "ws_floats", "counters", "chunk")

SHIM = r"""
#include "linear_plan.h"
extern "C" void plan(int rows, int k, int n, int mats, int drain, int sms, const int *clusters, long long *o) {
    const brk::LinearPlan p = brk::linear_plan_for(rows, k, n, mats, drain != 0, sms, [&](int s) { return clusters[s]; });
    const long long v[] = {p.pair, p.ranged, p.drain, p.cs, p.nt_kernel, p.nt, p.f_rows, p.half_cols, p.tiles_m, p.nk,
                           p.kb, p.stages, p.drain_steps, p.ctas, p.tiles, p.tiles_whole, p.range_units, p.range_extra,
                           (long long)p.ws_floats, (long long)p.counters, brk::linear_chunk(p.nt_kernel, p.drain)};
    for (unsigned i = 0; i < sizeof(v) / sizeof(v[0]); ++i) o[i] = v[i];
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(d / "plan.so"), str(d / "plan.cpp")],
                   check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))

    def call(rows, k, n, mats, drain, clusters=CLUSTERS[0]):
        out = (ctypes.c_longlong * len(FIELDS))()
        lib.plan(rows, k, n, mats, int(drain), SMS, (ctypes.c_int * 9)(*clusters), out)
        return dict(zip(FIELDS, out))
    return call


ROWS = sorted(set(range(5, 140)) | set(range(140, 2100, 13)) | {256, 257, 512, 513, 2048, 4096, 10000})
WIDTHS = [(10240, 2560), (4096, 2560), (2560, 2560), (2560, 10240), (1112, 7014), (6280, 3471), (5432, 4710), (8192, 8192),
          (1024, 4096), (72, 129), (8, 1), (2304, 9215)]


@pytest.mark.parametrize("clusters", CLUSTERS)
@pytest.mark.parametrize("k,n", WIDTHS)
def test_epilogue_warps_share_no_column(plan, k, n, clusters):
    """Where the accumulators are drained, the two epilogue warps of a lane quarter store their sums back in
    chunks: no column may be in a chunk of both.  And nothing is read past the accumulator, or written
    past a partial tile's slot."""
    for rows in ROWS:
        for mats, drain in ((1, True), (1, False), (2, False)):
            p = plan(rows, k, n, mats, drain, clusters)
            nt, half, ch = p["nt"], p["half_cols"], p["chunk"]
            assert nt % 16 == 0 and 16 <= nt <= p["nt_kernel"] <= 256
            if p["nt_kernel"] < 64:
                assert half == nt
                continue
            assert 2 * half >= nt and 2 * half <= p["nt_kernel"]
            ends = [col0 + -(-max(0, min(half, nt - col0)) // ch) * ch for col0 in (0, half)]
            assert max(ends) <= min(p["nt_kernel"], nt + 16)
            if drain and nt > half:
                assert ends[0] <= half, (rows, k, n, p)


@pytest.mark.parametrize("k,n", WIDTHS)
def test_every_k_step_once(plan, k, n):
    """The pieces of all workers (whole tiles wave by wave, then contiguous ranges of (tile, k step) units)
    cover every tile's k once."""
    for rows in ROWS[::7]:
        for mats, drain in ((1, True), (2, False)):
            p = plan(rows, k, n, mats, drain)
            ctas = 2 if p["pair"] else 1
            workers, nk, whole = p["ctas"] // (ctas * p["cs"]), p["nk"], p["tiles_whole"]
            assert p["ctas"] == workers * ctas * p["cs"] and workers >= 1
            assert p["tiles"] == -(-n // (p["f_rows"] * ctas)) * p["tiles_m"] and p["tiles_m"] * p["nt"] >= rows
            assert nk * p["kb"] * 64 >= k and (p["kb"] == 1 or k % 64 == 0)
            assert p["cs"] == 1 or (p["tiles"] == whole == workers and nk >= p["cs"])
            ranged = p["tiles"] - whole
            begin = lambda c: c * p["range_units"] + min(c, p["range_extra"])  # noqa: E731
            assert begin(workers) == ranged * nk and (ranged == 0 or p["range_units"] >= 1)
            assert p["counters"] == ranged * ctas and (p["ws_floats"] > 0) == (ranged > 0)
            if ranged:  # a tile's parts come from the workers whose ranges meet it, one slot of two each
                slot = (mats if not p["pair"] else 1) * p["nt"] + 16
                assert p["ws_floats"] >= p["ctas"] * 2 * slot * 128


B200 = (0, 148, 74, 45, 33, 26, 22, 15, 15)  # as the driver counts them for these kernels


def _form(p):
    ranged = p["tiles"] > p["tiles_whole"]
    cut = "cluster" if p["cs"] > 1 else "whole" if not ranged else "ranged after whole" if p["tiles_whole"] else "ranged"
    return "pair" if p["pair"] else "one", cut


def test_gpu_shapes_reach_every_form(plan):
    from test_gpu_linear_forms import GATE_UP, LINEAR
    for form, rows, k, n in LINEAR:
        p = plan(rows, k, n, 1, True, B200)
        assert _form(p) == form, (rows, k, n, p)
        # More than one accumulator set in a piece, and two warps to a lane quarter.
        steps = p["range_units"] if p["tiles"] > p["tiles_whole"] else p["nk"] // p["cs"]
        assert steps > p["drain_steps"] and p["nt_kernel"] >= 64, (rows, k, n, p)
        assert _form(plan(rows, k, n, 1, False, B200)) == form
    for form, rows, k, n in GATE_UP:
        assert _form(plan(rows, k, n, 2, False, B200)) == form, (rows, k, n, plan(rows, k, n, 2, False, B200))
    # Halves that are odd multiples of 16 when nothing is drained, one for each kernel that has two warps.
    halves = {(p["nt_kernel"], p["pair"]) for p in (plan(r, k, n, 1, False, B200) for _, r, k, n in LINEAR) if p["half_cols"] % 32}
    assert {(128, 0), (256, 0), (256, 1)} <= halves
    assert {f for f, *_ in LINEAR} | {("one", "ranged after whole")} >= {f for f, *_ in GATE_UP}
