"""The paged-cache entry points on the emulated wave64 machine, under ASan +
UBSan: the host code's checks and launch shapes and the kernels' own source,
against 64-bit oracles (paged_cases.py).

Pools hold NaN wherever no sequence has a position, so a read past a length,
of another page or of a masked place shows in the result; emulated buffers have
their exact sizes, so any access outside one stops the run.
"""
import os
import subprocess

import numpy as np
import pytest

import paged_cases as P
from helpers import REPO

EMU = os.path.join(REPO, "tests", "hostemu")

pytestmark = pytest.mark.skipif(not os.path.exists("/opt/rocm/lib/llvm/bin/clang++"), reason="ROCm clang not available")


@pytest.fixture(scope="module")
def built():
    r = subprocess.run(["make", "-C", EMU, "-j8"], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    return True


GLOBAL, LOCAL = 5, 0


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv", [(8, 4), (4, 1), (2, 2)])
def test_prefill_packed(built, tmp_path, hq, hkv, bf16):
    """Ragged prompts, one of them empty, one a single token, histories that
    end inside a page, rows behind the last sequence."""
    r = P.EmuRunner(tmp_path, hq=hq, hkv=hkv, window=24)
    P.run_prefill(r, GLOBAL, [37, 0, 1, 20], [37, 5, 50, 61], 16, bf16, padding=3)
    P.run_prefill(r, LOCAL, [19, 40], [60, 40], 32, bf16, seed=1, label="local")
    r.done()


def test_prefill_bad_tables_and_lengths(built, tmp_path):
    """Pages outside the pool are left out, a sequence shorter than its rows
    gives zeros to the rows before it, a length past its table is cut."""
    r = P.EmuRunner(tmp_path, hq=2, hkv=1, window=40)
    P.run_prefill(r, GLOBAL, [5, 9, 7], [50, 33, 7], 16, False, bad=[(0, 1, -1), (1, 0, 999), (1, 1, -7), (1, 2, 1 << 30)], label="bad pages")
    P.run_prefill(r, LOCAL, [12, 3], [5, 0], 16, False, seed=2, label="short")
    P.run_prefill(r, GLOBAL, [4], [1000], 16, True, seed=3, bad=[(0, j, -1) for j in range(60)], label="mostly absent")
    r.done()


def test_prefill_split_keys(built, tmp_path):
    """Few blocks over many keys: parts and their merge (256 emulated CUs)."""
    r = P.EmuRunner(tmp_path, hq=2, hkv=1, window=400, max_context=1024)
    P.run_prefill(r, GLOBAL, [3, 40], [900, 700], 64, False, label="parts")
    P.run_prefill(r, LOCAL, [33], [800], 16, True, seed=5, label="parts, local")
    out = r.done()
    assert "paged_prefill_merge_kernel" in out


@pytest.mark.parametrize("bf16", [False, True])
def test_scales(built, tmp_path, bf16):
    """Values far from 1: the block exponents keep their precision."""
    r = P.EmuRunner(tmp_path, hq=2, hkv=1)
    for i, (qs, ks) in enumerate([(2e6, 1e-6), (1e-9, 3e8), (0.0, 1.0)]):
        P.run_prefill(r, GLOBAL, [6], [45], 16, bf16, seed=i, scale=qs, kv_scale=ks, label=f"q {qs} kv {ks}")
    r.done()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv", [(8, 4), (4, 1), (2, 2)])
def test_decode(built, tmp_path, hq, hkv, bf16):
    r = P.EmuRunner(tmp_path, hq=hq, hkv=hkv, window=30)
    P.run_decode(r, GLOBAL, [1] * 5, [0] * 5, [1, 2, 33, 70, 16], 16, bf16, groups=False)
    P.run_decode(r, GLOBAL, [3, 1, 2], [40, 9, 0], [1, 5, 30, 3, 8, 2], 16, bf16, seed=1, label="groups")
    P.run_decode(r, LOCAL, [3, 2], [40, 17], [1, 50, 12, 3, 20], 16, bf16, seed=2, label="groups, local")
    r.done()


def test_decode_edges(built, tmp_path):
    """Sequences without a key, prefixes longer than a member, absent pages,
    more members than one block of rows holds, long tails cut into chunks."""
    r = P.EmuRunner(tmp_path, hq=4, hkv=1, window=64, max_context=1024)
    P.run_decode(r, GLOBAL, [1, 1, 1], [0, 0, 0], [0, 7, 0], 16, False, groups=False, label="empty")
    P.run_decode(r, GLOBAL, [20], [35], list(range(1, 21)), 16, False, seed=1, label="many members")
    P.run_decode(r, LOCAL, [20], [90], [1 + 9 * i for i in range(20)], 32, True, seed=4, label="many members, local")
    P.run_decode(r, GLOBAL, [2], [64], [900, 0], 16, False, seed=2, label="long tail, none")
    P.run_decode(r, GLOBAL, [2, 1], [30, 0], [40, 3, 60], 16, False, seed=3, bad=[(0, 3, -1), (2, 1, 77), (2, 0, -9)], label="absent")
    r.done()


def test_decode_malformed_groups(built, tmp_path):
    """Group bounds that overlap or run backwards stay inside the buffers."""
    r = P.EmuRunner(tmp_path, hq=2, hkv=1)
    rng = np.random.default_rng(0)
    lens, ps = [40, 50, 33, 20], 16
    table = P.tables_for(rng, lens, ps, 16)
    pool = P.Pool(rng, 1, 16, 1, ps, False, first_layer=GLOBAL)
    pool.fill(rng, table, lens)
    q = rng.standard_normal((4, 2, P.D)).astype(np.float32)
    r.pool(pool)
    r.seqs(0, lens, table)
    for groups in [([0, 9, -4, 4], [30, 1 << 30, 20]), ([3, 0, 4, 0], [5, 6, 7]), ([-5, 4, 0, 4], [-3, 33, 20])]:
        r.decode(GLOBAL, 0, groups, q, lambda out: None)
    r.prefill(GLOBAL, 0, [0, 3, 1, 9, 2], q, lambda out: None)
    r.prefill(GLOBAL, 0, [-7, 2, 2, -1, 1 << 30], q, lambda out: None)
    r.done()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv", [(8, 4), (4, 1), (3, 3)])
def test_write(built, tmp_path, hq, hkv, bf16):
    r = P.EmuRunner(tmp_path, hq=hq, hkv=hkv, max_context=128)
    P.run_write(r, LOCAL, [5, 0, 1, 17], [21, 4, 40, 17], 16, bf16, padding=2)
    P.run_write(r, GLOBAL - 1, [3, 4], [90, 4], 32, bf16, norm=False, seed=1, pool_kw=dict(order="pages", pad=8), label="no norm")
    P.run_write(r, LOCAL, [1] * 70, list(range(1, 71)), 16, bf16, seed=2, label="steps")
    r.done()


def test_write_edges(built, tmp_path):
    """Positions outside the context or below 0 and absent pages write nothing."""
    r = P.EmuRunner(tmp_path, hq=2, hkv=1, max_context=40)
    P.run_write(r, LOCAL, [6, 9], [45, 4], 16, False, label="outside")
    P.run_write(r, LOCAL, [20, 3], [20, 30], 16, True, seed=1, bad=[(0, 0, -1), (1, 1, 500)], label="absent")
    P.run_write(r, LOCAL, [0, 0, 2] + [0] * 90 + [3], [0, 5, 2] + [1] * 90 + [3], 16, False, seed=2, label="empty ones")
    r.done()


def test_fork(built, tmp_path):
    r = P.EmuRunner(tmp_path, hq=2, hkv=2)
    # beams: one parent twice, one ends, one slot falls empty
    _, _, st, copies = P.run_fork(r, [20, 33, 16, 7], [0, 0, 3, -1, 1], [1, 1, 1, 1, 0], 16, 16)
    assert len(copies) == 1 and st[1] == 0
    # a full page is shared, growth is a new page; the untouched one keeps its partial page, so growers copy
    P.run_fork(r, [32, 20], [0, 0, 1, 1, 1], [1, 17, 0, 5, 40], 16, 24, bf16=True, seed=1, stride=6, label="mixed")
    # rollback, to nothing too; a parent out of range
    P.run_fork(r, [40, 20, 9], [0, 1, 2, 7], [-10, -40, -9, 3], 16, 12, seed=2, label="rollback")
    # in place, identity
    P.run_fork(r, [5, 16, 31], [0, 1, 2], [1, 1, 1], 16, 9, seed=3, alias=True, label="step")
    P.run_fork(r, [5, 16, 31], [0, 1, 2], [0, 0, 0], 16, 9, seed=3, null=("parent", "add"), label="identity")
    r.done()


def test_fork_shortage_and_holds(built, tmp_path):
    r = P.EmuRunner(tmp_path, hq=1, hkv=1)
    # pages run out for the later ones; a table row is too short for one
    _, _, st, _ = P.run_fork(r, [30, 30], [0, 0, 1, 1], [1, 1, 40, 3], 16, 6, stride=4, label="short")
    assert st[1] > 0
    P.run_fork(r, [30, 30], [0, 1], [40, 2], 16, 9, seed=1, stride=4, label="row")
    held = np.zeros(20, np.int32)
    held[[0, 1, 5, 19]] = 1
    P.run_fork(r, [20, 40], [0, 1, 1], [3, 30, 1], 16, 20, held=held, seed=2, stride=8, label="held")
    # a held tail page, and entries outside the pool, in front and last
    P.run_fork(r, [20, 40, 18], [0, 1, 2], [3, 30, 5], 16, 20, held=held, seed=3, stride=8, bad=[(0, 1, 5), (1, 0, -3), (2, 1, 1 << 20)],
               label="held tail")
    # shared pages already
    P.run_fork(r, [36, 40, 33], [2, 0, 1, 1], [1, 0, 2, 9], 16, 20, seed=4, shared=[(0, 3, 2)], label="shared")
    # more sequences than one pass of the plan looks at, and pools past a wave's run
    n = 1100
    rng = np.random.default_rng(5)
    P.run_fork(r, list(rng.integers(0, 30, 40)), list(rng.integers(-1, 41, n)), list(rng.integers(-3, 9, n)), 16, 1000, seed=6, layers=1,
               stride=3, label="many")
    r.done()


@pytest.mark.parametrize("kw", [dict(order="pages"), dict(pad=16), dict(order="pages", pad=8)])
def test_fork_and_compact_strides(built, tmp_path, kw):
    r = P.EmuRunner(tmp_path, hq=2, hkv=2)
    P.run_fork(r, [20, 33], [0, 0, 1, 1], [1, 2, 1, 0], 16, 12, bf16=True, pool_kw=kw)
    P.run_compact(r, [20, 33, 16], 16, 12, pool_kw=kw)
    r.done()


def test_compact(built, tmp_path):
    r = P.EmuRunner(tmp_path, hq=2, hkv=1)
    P.run_compact(r, [20, 33, 0, 16, 1], 16, 30)
    P.run_compact(r, [20, 33], 16, 30, bf16=True, seed=1, alias=True, label="in place")
    P.run_compact(r, [40, 40, 45], 16, 64, seed=2, shared=[(0, 3, 2)], label="shared")
    held = np.zeros(70, np.int32)
    held[[0, 3, 40, 69]] = 1
    P.run_compact(r, [40, 40, 45], 16, 70, held=held, seed=3, label="held")
    P.run_compact(r, [40, 40], 16, 20, seed=3, bad=[(0, 1, -1), (1, 2, 1 << 30)], label="absent")
    P.run_compact(r, [0, 0], 16, 20, seed=4, label="empty")
    P.run_compact(r, [16] * 300, 16, 1500, seed=5, layers=1, label="large")
    r.done()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layer", [GLOBAL, LOCAL])
def test_spoiled_keys(built, tmp_path, layer, bf16):
    """An infinity or a NaN reaches the rows that see it and no others."""
    r = P.EmuRunner(tmp_path, hq=4, hkv=2, window=32)
    P.run_spoiled_all(r, layer, bf16)
    r.done()


@pytest.mark.parametrize("bf16", [False, True])
def test_faint_keys(built, tmp_path, bf16):
    r = P.EmuRunner(tmp_path, hq=2, hkv=1, max_context=4096)
    P.run_faint(r, GLOBAL, bf16, keys=1500)
    r.done()


@pytest.mark.parametrize("seed", range(6))
def test_decode_few_cus(built, tmp_path, seed):
    """Batches of every make-up on 4 and 12 emulated CUs: chunks, second rounds,
    packs of short sequences, odd chunk lengths."""
    rng = np.random.default_rng(seed)
    hq, hkv = [(2, 1), (4, 2), (4, 1)][seed % 3]
    r = P.EmuRunner(tmp_path, env={"HOSTEMU_CUS": str([4, 12][seed % 2])}, hq=hq, hkv=hkv, window=int(rng.integers(20, 200)), max_context=2048)
    for i in range(3):
        members = [int(m) for m in rng.integers(1, 9, int(rng.integers(1, 6)))]
        prefix = [int(p) for p in rng.integers(0, 300, len(members))]
        tail = [int(t) for t in np.where(rng.random(sum(members)) < 0.7, rng.integers(0, 60, sum(members)), rng.integers(1, 400, sum(members)))]
        P.run_decode(r, [GLOBAL, LOCAL][int(rng.integers(2))], members, prefix, tail, 16, bool(rng.integers(2)), seed=seed * 10 + i,
                     groups=bool(i), label=f"few CUs {seed}.{i}")
    r.done()


@pytest.mark.parametrize("bf16", [False, True])
def test_serving_loop(built, tmp_path, bf16):
    r = P.EmuRunner(tmp_path, hq=4, hkv=2, window=24)
    P.run_serving(r, bf16, rounds=1)
    r.done()


def test_refusals(built, tmp_path):
    """What the host can see is refused, before anything is touched."""
    r = P.EmuRunner(tmp_path, hq=4, hkv=2)
    r.lines.append("paged_refusals")
    assert "attn_emu: refused" in r.done()


def test_fork_and_compact_sizes(built, tmp_path):
    """At and past what one launch counts by itself: 32 sequences, 4096 pages."""
    r = P.EmuRunner(tmp_path, hq=1, hkv=1)
    rng = np.random.default_rng(8)
    lens = [int(n) for n in rng.integers(0, 70, 20)]
    for i, n in enumerate([31, 32, 33, 70]):
        P.run_fork(r, lens, [int(p) for p in rng.integers(-1, 21, n)], [int(x) for x in rng.integers(-5, 30, n)], 16, 500, seed=i, stride=8,
                   layers=1, label=f"{n} children")
        P.run_compact(r, [int(x) for x in rng.integers(0, 70, n)], 16, 500, seed=i, layers=1, label=f"{n} sequences")
    for i, pages in enumerate([4096, 4097]):
        P.run_fork(r, [20, 33, 40], [0, 0, 1, 2, 2], [1, 1, 20, 1, 1], 16, pages, seed=i, layers=1, stride=5, bf16=True, label=f"{pages} pages")
        P.run_compact(r, [20, 33, 40], 16, pages, seed=i, layers=1, bf16=True, label=f"{pages} pages")
    out = r.done()
    for kernel in ("fork_small_kernel", "fork_plan_kernel", "compact_small_kernel", "compact_plan_kernel"):
        assert kernel in out


@pytest.mark.parametrize("seed", range(4))
def test_prefill_few_cus(built, tmp_path, seed):
    """Packed prompts of every make-up on 4 and 12 emulated CUs, where 128-row
    workgroups run: whole and part chunks, classes, blocks that are not cut."""
    rng = np.random.default_rng(40 + seed)
    hq, hkv = [(2, 1), (4, 2), (4, 1), (2, 2)][seed]
    r = P.EmuRunner(tmp_path, env={"HOSTEMU_CUS": str([4, 12][seed % 2])}, hq=hq, hkv=hkv, window=int(rng.integers(40, 200)), max_context=2048)
    for i in range(2):
        n = int(rng.integers(1, 6))
        q = [int(x) for x in rng.integers(0, 120, n)]
        hist = [int(x) for x in np.where(rng.random(n) < 0.5, 0, rng.integers(0, 500, n))]
        P.run_prefill(r, [GLOBAL, LOCAL][i], q, [a + b for a, b in zip(q, hist)], 16, bool(rng.integers(2)), seed=seed * 10 + i,
                      label=f"few CUs {seed}.{i}")
    out = r.done()
    assert "paged_prefill_merge_kernel" in out
