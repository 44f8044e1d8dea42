"""The paged-cache entry points on the GPU against 64-bit oracles
(paged_cases.py, which derives the tolerances): every head layout, page type and
size, lengths from nothing to thousands, spoiled tables, refusals, a serving
loop of all of them, and graph replays."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as P
from helpers import DeviceBuffer

pytestmark = pytest.mark.gpu

GLOBAL, LOCAL = 5, 0
HEADS = [(8, 4), (16, 8), (4, 1), (4, 4)]


@pytest.fixture
def run():
    made = []

    def make(**kw):
        made.append(P.GpuRunner(**kw))
        return made[-1]
    yield make
    for r in made:
        r.done()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_write(run, hq, hkv, bf16):
    r = run(hq=hq, hkv=hkv, max_context=400)
    P.run_write(r, LOCAL, [5, 0, 1, 117], [21, 4, 390, 117], 16, bf16, padding=2)
    P.run_write(r, GLOBAL - 1, [3, 4], [90, 4], 32, bf16, norm=False, seed=1, pool_kw=dict(order="pages", pad=8), label="no norm")
    P.run_write(r, LOCAL, [1] * 70, list(range(1, 71)), 64, bf16, seed=2, label="steps")
    P.run_write(r, LOCAL, [20, 9, 3], [20, 405, 1], 16, bf16, seed=3, bad=[(0, 0, -1), (1, 1, 500)], label="outside")
    P.run_write(r, LOCAL, [0, 0, 2] + [0] * 90 + [3], [0, 5, 2] + [1] * 90 + [3], 16, bf16, seed=4, label="empty ones")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_prefill(run, hq, hkv, bf16):
    r = run(hq=hq, hkv=hkv, window=100, max_context=1024)
    P.run_prefill(r, GLOBAL, [37, 0, 1, 120], [37, 5, 50, 261], 16, bf16, padding=3)
    P.run_prefill(r, LOCAL, [190, 40], [260, 40], 32, bf16, seed=1, label="local")
    P.run_prefill(r, GLOBAL, [5, 9, 7], [50, 33, 7], 16, bf16, seed=2, bad=[(0, 1, -1), (1, 0, 999), (1, 1, -7), (1, 2, 1 << 30)],
                  label="absent")
    P.run_prefill(r, LOCAL, [12, 3], [5, 0], 128, bf16, seed=3, label="short")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layer", [GLOBAL, LOCAL])
def test_prefill_long(run, layer, bf16):
    """Histories of thousands, and blocks enough to fill the chip."""
    r = run(window=1024, max_context=4096)
    P.run_prefill(r, layer, [3, 140], [3001, 2111], 64, bf16, label="history")
    r2 = run(hq=4, hkv=4, window=512)
    P.run_prefill(r2, layer, [300] * 14 + [1] * 30, [300] * 14 + list(range(1, 31)), 16, bf16, seed=1, label="many")


@pytest.mark.parametrize("bf16", [False, True])
def test_scales(run, bf16):
    r = run(hq=2, hkv=1)
    for i, (qs, ks) in enumerate([(2e6, 1e-6), (1e-9, 3e8), (0.0, 1.0)]):
        P.run_prefill(r, GLOBAL, [6], [45], 16, bf16, seed=i, scale=qs, kv_scale=ks, label=f"q {qs} kv {ks}")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_decode(run, hq, hkv, bf16):
    r = run(hq=hq, hkv=hkv, window=300, max_context=8192)
    P.run_decode(r, GLOBAL, [1] * 5, [0] * 5, [1, 2, 33, 700, 16], 16, bf16, groups=False)
    P.run_decode(r, GLOBAL, [3, 1, 2], [400, 9, 0], [1, 5, 300, 3, 8, 2], 16, bf16, seed=1, label="groups")
    P.run_decode(r, LOCAL, [3, 2], [400, 17], [1, 500, 12, 3, 20], 32, bf16, seed=2, label="groups, local")
    P.run_decode(r, GLOBAL, [70, 3], [135, 64], [1 + i % 50 for i in range(73)], 16, bf16, seed=3, label="many members")
    P.run_decode(r, GLOBAL, [2], [2000], [3000, 0], 64, bf16, seed=4, label="long")
    P.run_decode(r, GLOBAL, [1, 1, 1], [0, 0, 0], [0, 7, 0], 16, bf16, seed=5, groups=False, label="empty")
    P.run_decode(r, GLOBAL, [2, 1], [30, 0], [40, 3, 60], 16, bf16, seed=6, bad=[(0, 3, -1), (2, 1, 77), (2, 0, -9)], label="absent")


def test_decode_malformed_groups(run):
    """Group bounds and row offsets that overlap or run backwards stay inside the
    buffers, as on the emulated machine."""
    r = run(hq=2, hkv=1)
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


def test_many_sequences(run):
    """More sequences than a wave looks at in one go, most of them short."""
    r = run(hq=4, hkv=1, max_context=2048)
    n = 300
    P.run_decode(r, GLOBAL, [1] * n, [0] * n, [1 + (7 * i) % 40 for i in range(n)], 16, True, groups=False, label="300 sequences")
    P.run_decode(r, GLOBAL, [30] * 10, [20 + 3 * i for i in range(10)], [1 + (7 * i) % 40 for i in range(n)], 16, False, seed=1, label="10 groups")
    P.run_prefill(r, GLOBAL, [i % 3 for i in range(n)], [i % 3 + i % 20 for i in range(n)], 16, False, seed=2, label="300 prompts")


def test_fork(run):
    r = run(hq=2, hkv=2)
    _, _, st, copies = P.run_fork(r, [20, 33, 16, 7], [0, 0, 3, -1, 1], [1, 1, 1, 1, 0], 16, 16)
    assert len(copies) == 1 and st[1] == 0
    P.run_fork(r, [32, 20], [0, 0, 1, 1, 1], [1, 17, 0, 5, 40], 16, 24, bf16=True, seed=1, stride=6, label="mixed")
    P.run_fork(r, [40, 20, 9], [0, 1, 2, 7], [-10, -40, -9, 3], 16, 12, seed=2, label="rollback")
    P.run_fork(r, [5, 16, 31], [0, 1, 2], [1, 1, 1], 16, 9, seed=3, alias=True, label="step")
    P.run_fork(r, [5, 16, 31], [0, 1, 2], [0, 0, 0], 16, 9, seed=3, null=("parent", "add"), label="identity")
    P.run_fork(r, [20, 33, 16, 7], [3, 0, 0, 1], [1, 1, 1, 1], 16, 16, seed=4, alias=True, label="reordered in place")
    _, _, st, _ = P.run_fork(r, [30, 30], [0, 0, 1, 1], [1, 1, 40, 3], 16, 6, stride=4, label="short")
    assert st[1] > 0
    P.run_fork(r, [30, 30], [0, 1], [40, 2], 16, 9, seed=1, stride=4, label="row")
    held = np.zeros(20, np.int32)
    held[[0, 1, 5, 19]] = 1
    P.run_fork(r, [20, 40], [0, 1, 1], [3, 30, 1], 16, 20, held=held, seed=2, stride=8, label="held")
    P.run_fork(r, [20, 40, 18], [0, 1, 2], [3, 30, 5], 16, 20, held=held, seed=3, stride=8, bad=[(0, 1, 5), (1, 0, -3), (2, 1, 1 << 20)],
               label="held tail")
    P.run_fork(r, [36, 40, 33], [2, 0, 1, 1], [1, 0, 2, 9], 16, 20, seed=4, shared=[(0, 3, 2)], label="shared")
    rng = np.random.default_rng(5)
    P.run_fork(r, list(rng.integers(0, 90, 400)), list(rng.integers(-1, 401, 3000)), list(rng.integers(-3, 40, 3000)), 16, 5003, seed=6,
               layers=1, stride=9, label="many")


def test_fork_and_compact_sizes(run):
    """At and past what one launch counts by itself: 32 sequences, 4096 pages."""
    r = run(hq=1, hkv=1)
    rng = np.random.default_rng(8)
    lens = [int(n) for n in rng.integers(0, 70, 20)]
    for i, n in enumerate([31, 32, 33, 70]):
        P.run_fork(r, lens, [int(p) for p in rng.integers(-1, 21, n)], [int(x) for x in rng.integers(-5, 30, n)], 16, 500, seed=i, stride=8,
                   layers=1, label=f"{n} children")
        P.run_compact(r, [int(x) for x in rng.integers(0, 70, n)], 16, 500, seed=i, layers=1, label=f"{n} sequences")
    for i, pages in enumerate([4096, 4097]):
        P.run_fork(r, [20, 33, 40], [0, 0, 1, 2, 2], [1, 1, 20, 1, 1], 16, pages, seed=i, layers=1, stride=5, bf16=True, label=f"{pages} pages")
        P.run_compact(r, [20, 33, 40], 16, pages, seed=i, layers=1, bf16=True, label=f"{pages} pages")


def test_compact(run):
    r = run(hq=2, hkv=1)
    P.run_compact(r, [20, 33, 0, 16, 1], 16, 30)
    P.run_compact(r, [20, 33], 16, 30, bf16=True, seed=1, alias=True, label="in place", pool_kw=dict(order="pages", pad=8))
    P.run_compact(r, [40, 40, 45], 16, 64, seed=2, shared=[(0, 3, 2)], label="shared")
    held = np.zeros(70, np.int32)
    held[[0, 3, 40, 69]] = 1
    P.run_compact(r, [40, 40, 45], 16, 70, held=held, seed=3, label="held")
    P.run_compact(r, [40, 40], 16, 20, seed=3, bad=[(0, 1, -1), (1, 2, 1 << 30)], label="absent")
    P.run_compact(r, [0, 0], 16, 20, seed=4, label="empty")
    P.run_compact(r, [16] * 2000, 16, 9001, seed=5, layers=1, label="large")


def test_refusals(run):
    """What the host can see is refused with a message before anything is enqueued."""
    r = run(hq=4, hkv=2, layers=6)
    G, ctx = r.G, r.ctx
    A, T, O = 1 << 40, 1 << 42, 1 << 44      # never followed: each call is refused first

    def pages(**kw):
        d = dict(k=A, v=A, dtype=G.PAGE_F32, first_layer=0, num_layers=6, num_pages=8, page_size=16, page_stride=2 * 16 * 256,
                 layer_stride=8 * 2 * 16 * 256)
        d.update(kw)
        return G.Pages(**d)

    def seqs(**kw):
        d = dict(num_seqs=2, kv_len=A, page_table=T, table_stride=4)
        d.update(kw)
        return G.Seqs(**d)

    def batch(total=7, start=A, **kw):
        return G.Batch(seqs=seqs(**kw), total_q=total, q_start=start)

    def refused(f, *a):
        with pytest.raises(G.G3AttnError) as e:
            f(*a)
        assert e.value.rc == G.ERR_INVALID_ARG and str(e.value)
    for bad in (dict(k=None), dict(v=None), dict(dtype=2), dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(num_pages=0),
                dict(num_layers=0), dict(first_layer=-1), dict(page_stride=2 * 16 * 256 - 8), dict(page_stride=2 * 16 * 256 + 4),
                dict(layer_stride=8), dict(k=A + 4), dict(layer_stride=7 * 2 * 16 * 256)):
        refused(ctx.paged_prefill_device, 0, pages(**bad), batch(), A, O)
        refused(ctx.pages_compact_device, pages(**bad), seqs(), None, seqs())
    for layer, first in ((6, 0), (-1, 0), (0, 1), (5, 6)):
        refused(ctx.paged_prefill_device, layer, pages(first_layer=first), batch(), A, O)
    for bad in (dict(num_seqs=0), dict(num_seqs=4097), dict(kv_len=None), dict(page_table=None), dict(table_stride=0), dict(table_stride=1 << 21)):
        refused(ctx.paged_write_device, 0, pages(), batch(**bad), A, A, A, None, None, O)
        refused(ctx.paged_decode_device, 0, pages(), batch(2, None, **bad), None, A, O)
        refused(ctx.pages_fork_device, pages(), seqs(**bad), None, None, None, seqs())
        refused(ctx.pages_fork_device, pages(), seqs(), None, None, None, seqs(**bad))
    for b in (batch(-1), batch((1 << 24) + 1), batch(3, None), None):
        refused(ctx.paged_prefill_device, 0, pages(), b, A, O)
    for a in ((None, A, A, O), (A, None, A, O), (A, A, None, O), (A, A, A, None), (A + 4, A, A, O)):
        refused(ctx.paged_write_device, 0, pages(), batch(), *a[:3], None, None, a[3])
    refused(ctx.paged_write_device, 0, pages(), batch(), A, A, A, A, None, O)
    refused(ctx.paged_write_device, 0, pages(), batch(), A, A, A, A + 2, A, O)
    refused(ctx.paged_prefill_device, 0, pages(), batch(), None, O)
    refused(ctx.paged_prefill_device, 0, pages(), batch(), A, O + 8)
    refused(ctx.paged_decode_device, 0, pages(), batch(), None, A, O)
    refused(ctx.paged_decode_device, 0, pages(), batch(2, None), G.Prefixes(num_groups=3, group_start=A, prefix_len=A), A, O)
    refused(ctx.paged_decode_device, 0, pages(), batch(2, None), G.Prefixes(num_groups=1, group_start=None, prefix_len=A), A, O)
    refused(ctx.paged_decode_device, 0, pages(), batch(2, None), G.Prefixes(num_groups=-1, group_start=A, prefix_len=A), A, O)
    refused(ctx.pages_fork_device, pages(), seqs(), None, None, None, seqs(table_stride=5))
    refused(ctx.pages_compact_device, pages(), seqs(), None, seqs(num_seqs=3))
    assert G.lib().g3attn_paged_prefill_device(None, 0, C.byref(pages()), C.byref(batch()), A, A) == G.ERR_INVALID_ARG
    ctx.paged_prefill_device(0, pages(), batch(0), None, None)      # nothing to do
    with G.Context(G.default_config(num_layers=1, max_context=16), 16, defer_rope=True) as bare:
        refused(bare.paged_write_device, 0, pages(num_layers=1, page_stride=4 * 16 * 256), batch(), A, A, A, None, None, O)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layer", [GLOBAL, LOCAL])
def test_spoiled_keys(run, layer, bf16):
    """An infinity or a NaN reaches the rows that see it and no others."""
    P.run_spoiled_all(run(hq=4, hkv=2, window=32), layer, bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_faint_keys(run, bf16):
    P.run_faint(run(hq=4, hkv=2, max_context=8192), GLOBAL, bf16, keys=5000)


@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("seed", range(3))
def test_decode_make_up(run, seed, hq, hkv):
    """Runs of members, prefixes and tails of many lengths together."""
    rng = np.random.default_rng(100 * seed + hq + hkv)
    r = run(hq=hq, hkv=hkv, window=int(rng.integers(20, 600)), max_context=8192)
    for i in range(3):
        members = [int(m) for m in rng.integers(1, 40, int(rng.integers(1, 7)))]
        n = sum(members)
        prefix = [int(p) for p in rng.integers(0, 1500, len(members))]
        tail = [int(t) for t in np.where(rng.random(n) < 0.8, rng.integers(0, 140, n), rng.integers(1, 1200, n))]
        P.run_decode(r, [GLOBAL, LOCAL][int(rng.integers(2))], members, prefix, tail, [16, 64][int(rng.integers(2))], bool(rng.integers(2)),
                     seed=seed * 10 + i, groups=bool(i), label=f"make-up {seed}.{i}")


@pytest.mark.parametrize("bf16", [False, True])
def test_serving_loop(run, bf16):
    P.run_serving(run(hq=8, hkv=4, window=24), bf16)


class FarPages(P.GpuRunner):
    """The pool's pages 2^28 elements apart, K and V of both layers beside each
    other: byte and element offsets beyond 32 bits."""

    def pool(self, p):
        rows = p.hkv * p.ps * P.D
        elem = 2 if p.bf16 else 4
        self.p, stride = p, 1 << 28
        buf = DeviceBuffer((p.pages - 1) * stride * elem + 2 * p.layers * rows * elem)
        self.keep.append(buf)
        self.pages = self.G.Pages(k=buf.ptr, v=buf.ptr + rows * elem, dtype=int(p.bf16), first_layer=p.first, num_layers=p.layers,
                                  num_pages=p.pages, page_size=p.ps, page_stride=stride, layer_stride=2 * rows)


@pytest.mark.parametrize("bf16", [False, True])
def test_far_pages(bf16):
    r = FarPages(hq=4, hkv=2, window=24)
    try:
        P.run_serving(r, bf16, seed=3, rounds=1)
    finally:
        r.done()


class Graphs:
    """Capture and replay on a context's stream."""

    def __init__(self, ctx):
        self.hip, vp = DeviceBuffer.hip(), C.c_void_p
        self.hip.hipStreamBeginCapture.argtypes = [vp, C.c_int]
        self.hip.hipStreamEndCapture.argtypes = [vp, C.POINTER(vp)]
        self.hip.hipGraphInstantiate.argtypes = [C.POINTER(vp), vp, vp, vp, C.c_size_t]
        self.hip.hipGraphLaunch.argtypes = [vp, vp]
        for f in ("hipGraphExecDestroy", "hipGraphDestroy"):
            getattr(self.hip, f).argtypes = [vp]
        self.ctx, self.stream, self.graph, self.exe = ctx, vp(ctx.stream()), vp(), vp()

    def capture(self, calls):
        assert self.hip.hipStreamBeginCapture(self.stream, 2) == 0        # hipStreamCaptureModeRelaxed
        try:
            calls()
        finally:
            assert self.hip.hipStreamEndCapture(self.stream, C.byref(self.graph)) == 0

    def replay(self):
        if not self.exe:
            assert self.hip.hipGraphInstantiate(C.byref(self.exe), self.graph, None, None, 0) == 0
        assert self.hip.hipGraphLaunch(self.exe, self.stream) == 0

    def close(self):
        if self.exe:
            self.hip.hipGraphExecDestroy(self.exe)
        if self.graph:
            self.hip.hipGraphDestroy(self.graph)


@pytest.mark.parametrize("bf16", [False, True])
def test_graph_replays(run, bf16):
    """A step of a serving loop (every sequence grows by a token, is written,
    decodes behind its shared prefix and sees its last rows again as a packed
    prompt; then the pool is compacted) captured once and replayed, against the
    same step called eagerly on a second pool.  Between replays the context
    does other work in the same scratch memory.  The order of every sum is
    fixed, so the results are the same bits."""
    r = run(hq=8, hkv=4, window=40)
    rng = np.random.default_rng(5)
    ps, pages, lens, prefix = 16, 48, [100, 70, 66, 31], [64, 0]
    first = [0, 3, 4]
    B, width = len(lens), 12
    table = P.tables_for(rng, lens, ps, pages, stride=width, shared=[(0, 3, 4)])
    pool = P.Pool(rng, 1, pages, r.hkv, ps, bf16, first_layer=GLOBAL, fill=0.0)
    pool.fill(rng, table, lens)
    G, ctx = r.G, r.ctx
    new = [r.buf(np.zeros((B, h, P.D), np.float32)) for h in (r.hq, r.hkv, r.hkv)]
    qn, kn = (r.put(P.to_bf16(rng.standard_normal(P.D) * 0.3)) for _ in range(2))
    groups = G.Prefixes(num_groups=2, group_start=r.put(np.asarray(first, np.int32)), prefix_len=r.put(np.asarray(prefix, np.int32)))
    add = r.put(np.ones(B, np.int32))
    rows = r.put(np.asarray([0, 2, 2, 4, 4], np.int32))        # two rows of the first, two of the third

    class Server:
        def __init__(self):
            self.k, self.v = r.buf(pool.pack(pool.k)), r.buf(pool.pack(pool.v))
            self.n, self.t = r.buf(np.asarray(lens, np.int32)), r.buf(table)
            self.q, self.o, self.o2 = (r.buf(np.zeros((B, r.hq, P.D), np.float32)) for _ in range(3))
            self.status = r.buf(np.zeros(4, np.int32))
            self.pages = G.Pages(k=self.k.ptr, v=self.v.ptr, dtype=int(bf16), first_layer=GLOBAL, num_layers=1, num_pages=pages, page_size=ps,
                                 page_stride=pool.page_stride, layer_stride=pool.layer_stride)
            self.seqs = G.Seqs(num_seqs=B, kv_len=self.n.ptr, page_table=self.t.ptr, table_stride=width)

        def step(self):
            one = G.Batch(seqs=self.seqs, total_q=B, q_start=None)
            ctx.pages_fork_device(self.pages, self.seqs, None, add, None, self.seqs, self.status.ptr)
            ctx.paged_write_device(GLOBAL, self.pages, one, *(x.ptr for x in new), qn, kn, self.q.ptr)
            ctx.paged_decode_device(GLOBAL, self.pages, one, groups, self.q.ptr, self.o.ptr)
            ctx.paged_prefill_device(GLOBAL, self.pages, G.Batch(seqs=self.seqs, total_q=B, q_start=rows), self.q.ptr, self.o2.ptr)
            ctx.pages_compact_device(self.pages, self.seqs, None, self.seqs, self.status.ptr + 8)

        def state(self):
            ctx.synchronize()
            return [b.download(np.uint8, b.nbytes) for b in (self.n, self.t, self.status, self.q, self.o, self.o2, self.k, self.v)]

    eager, graphed, other = Server(), Server(), Server()
    other.step()                       # the scratch memory grows here
    g = Graphs(ctx)
    try:
        g.capture(graphed.step)
        for rep in range(5):
            for b, h in zip(new, (r.hq, r.hkv, r.hkv)):
                b.upload(rng.standard_normal((B, h, P.D)).astype(np.float32))
            g.replay()
            if rep < 3:
                other.step()
            eager.step()
            for i, (a, b) in enumerate(zip(graphed.state(), eager.state())):
                assert np.array_equal(a, b), f"replay {rep}, buffer {i}"
    finally:
        g.close()
    assert list(eager.n.download(np.int32, B)) == [n + 5 for n in lens]


def test_scratch_does_not_grow_under_capture(run):
    """Refused with a message while the stream is captured, and fine after."""
    r = run(hq=8, hkv=4, max_context=2048)
    n = 200
    q = np.zeros((n, r.hq, P.D), np.float32)
    lens = [600] * n
    table = np.zeros((n, 38), np.int32)
    pool = P.Pool(np.random.default_rng(0), 1, 1, r.hkv, 16, False, first_layer=GLOBAL, fill=1.0)
    r.pool(pool)
    r.seqs(0, lens, table)
    qb, out = r.buf(q), r.buf(q)
    g = Graphs(r.ctx)

    def refused():
        with pytest.raises(r.G.G3AttnError) as e:
            r.ctx.paged_decode_device(GLOBAL, r.pages, r.batch(0, n, None), None, qb.ptr, out.ptr)
        assert e.value.rc == r.G.ERR_INVALID_ARG and "captured" in str(e.value)
    try:
        g.capture(refused)
    finally:
        g.close()
    r.decode(GLOBAL, 0, None, q, lambda o: np.testing.assert_allclose(o, 1.0, rtol=1e-5))
