"""What the paged-cache tests share: 64-bit oracles of the operators, pools
filled with NaN outside what sequences hold, and two runners with one
interface, the emulated machine of tests/hostemu (a script) and the GPU.

Tolerances, derived from the arithmetic:
- attention (rel: 2-norm of the difference over the result's).  Operands keep
  22 bits and a product drops lo.lo: three errors of at most 2^-22 each, so a
  score of standard deviation s (2 here) is off by about 2^-22 s = 5e-7; its 256
  fp32 additions add sqrt(256 / 3) 2^-24 s = 1.1e-6, the probabilities and
  values as much again on a smaller scale.  Together 2e-6; four times that is
  allowed, 8e-6.  One lost lo plane costs 2^-12.8 = 1.4e-4.
- writes (elementwise): sums of squares, root, division and three products are
  at most 20 half steps of 2^-24 on each of a pair (a, b), whose rotation
  mixes them: 20 2^-24 hypot(a, b); a bf16 page adds its half step, 2^-8.
"""
import os
import subprocess

import numpy as np

from helpers import REPO, DeviceBuffer, g3attn

D = 256
REL = 8e-6
EMU_EXE = os.path.join(REPO, "tests", "hostemu", "_build", "attn_emu")


def to_bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (np.asarray(u, np.uint16).astype(np.uint32) << 16).view(np.float32)


def rope_table(n, theta):
    a = np.arange(n)[:, None] * theta ** (-np.arange(D // 2) * 2.0 / D)[None]
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


# ------------------------------------------------------------------ the pool

class Pool:
    """Pages [layer][page][head][row][256] on the host, as fp32 values, and the
    memory they lie in: dense, padded pages, or page after page."""

    def __init__(self, rng, layers, pages, hkv, ps, bf16, first_layer=0, order="layers", pad=0, fill=np.nan):
        self.layers, self.pages, self.hkv, self.ps, self.bf16, self.first = layers, pages, hkv, ps, bf16, first_layer
        rows = hkv * ps * D
        if order == "layers":
            self.page_stride = rows + pad
            self.layer_stride = self.page_stride * pages
        else:
            self.layer_stride = rows + pad
            self.page_stride = self.layer_stride * layers
        self.size = layers * pages * (rows + pad)
        self.k = np.full((layers, pages, hkv, ps, D), fill, np.float32)
        self.v = np.full((layers, pages, hkv, ps, D), fill, np.float32)

    def _at(self):
        i = np.arange(self.layers)[:, None] * self.layer_stride + np.arange(self.pages)[None] * self.page_stride
        return i[..., None] + np.arange(self.hkv * self.ps * D)

    def pack(self, x):
        m = np.full(self.size, 7777.0, np.float32)
        m[self._at()] = x.reshape(self.layers, self.pages, -1)
        return to_bf16(m) if self.bf16 else m

    def unpack(self, m):
        m = from_bf16(m) if self.bf16 else m
        at = self._at()
        rest = np.ones(self.size, bool)
        rest[at] = False
        assert np.all(m[rest] == (from_bf16(to_bf16(np.float32(7777.0))) if self.bf16 else 7777.0)), "padding was written"
        return m[at].reshape(self.k.shape)

    def rows(self, layer, table, n, which):
        """[n][hkv][D] of positions 0 .. n - 1; NaN where the page is outside the pool."""
        x = getattr(self, which)[layer - self.first]
        out = np.full((n, self.hkv, D), np.nan, np.float64)
        for p in range(n):
            page = table[p // self.ps]
            if 0 <= page < self.pages:
                out[p] = x[page, :, p % self.ps]
        return out

    def fill(self, rng, tables, lens, scale=1.0):
        """Random values where sequences have positions."""
        seen = set()
        for t, n in zip(tables, lens):
            for p in range(min(int(n), len(t) * self.ps)):
                page = t[p // self.ps]
                if 0 <= page < self.pages and (page, p % self.ps) not in seen:
                    seen.add((page, p % self.ps))
                    for x in (self.k, self.v):
                        x[:, page, :, p % self.ps] = self.round(rng.standard_normal((self.layers, self.hkv, D)) * scale)

    def round(self, x):
        return from_bf16(to_bf16(x)) if self.bf16 else np.asarray(x, np.float32)


def tables_for(rng, lens, ps, pages, stride=None, shared=()):
    """Page tables of distinct pages in random order; shared = [(first, members,
    full pages)]."""
    need = [-(-int(n) // ps) for n in lens]
    stride = stride or max(need + [1]) + 1
    order = list(rng.permutation(pages))
    t = np.full((len(lens), stride), -1, np.int32)
    lead = {b: (f, c) for f, m, c in shared for b in range(f + 1, f + m)}
    for b, n in enumerate(need):
        f, c = lead.get(b, (b, 0))
        c = min(c, n)
        t[b, :c] = t[f, :c]
        for j in range(c, n):
            t[b, j] = order.pop()
    return t


# ------------------------------------------------------------------ oracles

def attention(q, k, v, ok, pos, window):
    """q [Hq][D] at pos, k / v [n][Hkv][D], ok [n]: what the query gives."""
    group = q.shape[0] // k.shape[1]
    lo = max(0, pos + 1 - window)
    hi = min(pos + 1, len(k))
    out = np.zeros(q.shape)
    keep = [j for j in range(lo, hi) if ok[j]]
    if not keep:
        return out
    for h in range(q.shape[0]):
        s = k[keep, h // group] @ q[h].astype(np.float64) / 16.0
        p = np.exp(s - s.max())
        out[h] = p @ v[keep, h // group] / p.sum()
    return out


def packed_attention(pool, layer, window, table, lens, q_start, q):
    out = np.full(q.shape, np.nan)
    for b in range(len(lens)):
        n = min(max(int(lens[b]), 0), table.shape[1] * pool.ps)
        k, v = pool.rows(layer, table[b], n, "k"), pool.rows(layer, table[b], n, "v")
        ok = [0 <= table[b][j // pool.ps] < pool.pages for j in range(n)]
        m = q_start[b + 1] - q_start[b]
        for i in range(m):
            out[q_start[b] + i] = attention(q[q_start[b] + i], k, v, ok, n - m + i, window)
    return out


def norm_rope(x, gain, table, pos, eps=1e-6):
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + from_bf16(gain).astype(np.float64))
    c, s = table[pos, :, 0].astype(np.float64), table[pos, :, 1].astype(np.float64)
    a, b = x[..., :128], x[..., 128:]
    y = np.concatenate([a * c - b * s, a * s + b * c], -1)
    h = np.hypot(a, b)
    return y, np.concatenate([h, h], -1)


def fork(table, lens, parent, add, held, ps, pages):
    """(table, lens, status, copies [(src, dst, rows)]) by the header's words."""
    width = table.shape[1]
    B = len(parent)
    old, want, full, kept, refused = [], [], [], [], [False] * B
    rows = []
    for b in range(B):
        real = 0 <= parent[b] < len(lens)
        o = min(max(int(lens[parent[b]]), 0), width * ps) if real else 0
        w = max(o + int(add[b]), 0) if real else 0
        if w > width * ps:
            w, refused[b] = o, True
        old.append(o)
        want.append(w)
        kept.append(-(-min(o, w) // ps))
        full.append(-(-w // ps))
        rows.append([int(x) for x in table[parent[b]]] if real else [])
    ref = [1 if held is not None and held[p] else 0 for p in range(pages)]
    for b in range(B):
        for p in rows[b][:kept[b]]:
            if 0 <= p < pages:
                ref[p] += 1
    tails = {}
    for b in range(B):
        if want[b] > old[b] and old[b] % ps:
            p = rows[b][old[b] // ps]
            if 0 <= p < pages:
                tails.setdefault(p, []).append(b)
    copies_of = {}
    for p, who in tails.items():
        for b in who:
            if not (b == who[0] and len(who) == ref[p]):
                copies_of[b] = p
    free = [p for p in range(pages) if ref[p] == 0]
    at, given, out, lens_out, copies = 0, 0, np.full((B, width), -1, np.int32), [], []
    for b in range(B):
        need = full[b] - kept[b] + (b in copies_of)
        mine = range(at, at + need)
        at += need
        if refused[b] or (need and mine[-1] >= len(free)):
            refused[b] = True
            want[b], full[b] = old[b], kept[b]
            copies_of.pop(b, None)
            mine = []
        new = [free[i] for i in mine]
        given += len(new)
        r = rows[b][:kept[b]]
        if b in copies_of:
            dst = new.pop(0)
            copies.append((copies_of[b], dst, old[b] % ps))
            r[old[b] // ps] = dst
        r += new
        out[b, :len(r)] = r
        lens_out.append(want[b])
    used = sum(x > 0 for x in ref) + given
    return out, np.array(lens_out, np.int32), [used, sum(refused)], copies


def compact(table, lens, held, ps, pages):
    width = table.shape[1]
    lens = np.array([min(max(int(n), 0), width * ps) for n in lens], np.int32)
    hold = {p for p in range(pages) if held is not None and held[p]}
    live = set(hold)
    for t, n in zip(table, lens):
        live |= {int(p) for p in t[:-(-int(n) // ps)] if 0 <= p < pages}
    used = len(live)
    src = [p for p in sorted(live) if p >= used and p not in hold]
    dst = [p for p in range(used) if p not in live][:len(src)]
    to = dict(zip(src, dst))
    out = np.full_like(table, -1)
    for b, n in enumerate(lens):
        for j in range(-(-int(n) // ps)):
            out[b, j] = to.get(int(table[b, j]), int(table[b, j]))
    return out, lens, [used, len(src)], list(zip(src, dst))


# ------------------------------------------------------------------ runners

def check_close(got, want, label, rel=REL):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.all(np.isfinite(got)), f"{label}: not finite"
    norm = np.linalg.norm(want)
    err = np.linalg.norm(got - want) / norm if norm else np.linalg.norm(got)
    worst = np.max(np.abs(got - want) / np.maximum(np.abs(want), norm / np.sqrt(want.size))) if norm else np.max(np.abs(got), initial=0.0)
    print(f"[paged] {label}: rel {err:.2e} max {worst:.2e}", flush=True)
    assert err <= rel and worst <= 40 * rel, f"{label}: rel {err:.2e} max {worst:.2e}"


class Runner:
    """Calls in order; each gives its outputs to a check, at once or when the
    script has run."""

    def __init__(self, hq=8, hkv=4, layers=6, window=64, max_context=512, theta=(1e4, 1e6)):
        self.hq, self.hkv, self.layers, self.window, self.max_context = hq, hkv, layers, window, max_context
        self.tables = {False: rope_table(max_context, theta[0]), True: rope_table(max_context, theta[1])}

    def span(self, layer):
        return 1 << 40 if (layer + 1) % 6 == 0 else self.window

    def rope(self, layer):
        return self.tables[(layer + 1) % 6 == 0]


class EmuRunner(Runner):
    def __init__(self, tmp, env=None, **kw):
        super().__init__(**kw)
        self.dir, self.n, self.lines, self.after, self.env = str(tmp), 0, [], [], env or {}
        rl, rg = self.put(self.tables[False]), self.put(self.tables[True])
        self.lines.append(f"create {self.hq} {self.hkv} {self.max_context} {self.window} {self.layers} 1e-6 {rl} {rg}")

    def name(self):
        self.n += 1
        return f"f{self.n}.bin"

    def put(self, a):
        if a is None:
            return "-"
        f = self.name()
        np.ascontiguousarray(a).tofile(os.path.join(self.dir, f))
        return f

    def get(self, f, dtype, shape):
        return np.fromfile(os.path.join(self.dir, f), dtype).reshape(shape)

    def pool(self, p):
        self.p = p
        self.lines.append(f"pool {int(p.bf16)} {p.first} {p.layers} {p.pages} {p.ps} {p.page_stride} {p.layer_stride} "
                          f"{self.put(p.pack(p.k))} {self.put(p.pack(p.v))}")

    def seqs(self, slot, lens, table):
        self.lines.append(f"seqs {slot} {len(lens)} {table.shape[1]} {self.put(np.asarray(lens, np.int32))} "
                          f"{self.put(np.asarray(table, np.int32))}")

    def pool_out(self, check):
        k, v = self.name(), self.name()
        dt = np.uint16 if self.p.bf16 else np.float32
        p = self.p
        self.lines.append(f"pool_out {k} {v}")
        self.after.append(lambda: check(p.unpack(self.get(k, dt, -1)), p.unpack(self.get(v, dt, -1))))

    def seqs_out(self, slot, shape, check):
        n, t = self.name(), self.name()
        self.lines.append(f"seqs_out {slot} {n} {t}")
        self.after.append(lambda: check(self.get(n, np.int32, -1), self.get(t, np.int32, shape)))

    def write(self, layer, slot, q_start, Q, K, V, qn, kn, check):
        out = self.put(np.full(Q.shape, 4444.0, np.float32))
        self.lines.append(f"paged_write {layer} {slot} {len(Q)} {self.put(_i32(q_start))} {self.put(Q)} {self.put(K)} {self.put(V)} "
                          f"{self.put(qn)} {self.put(kn)} {out}")
        self.after.append(lambda: check(self.get(out, np.float32, Q.shape)))

    def prefill(self, layer, slot, q_start, q, check):
        out = self.put(np.full(q.shape, 4444.0, np.float32))
        self.lines.append(f"paged_prefill {layer} {slot} {len(q)} {self.put(_i32(q_start))} {self.put(q)} {out}")
        self.after.append(lambda: check(self.get(out, np.float32, q.shape)))

    def decode(self, layer, slot, groups, q, check):
        out = self.put(np.full(q.shape, 4444.0, np.float32))
        g = f"{len(groups[1])} {self.put(_i32(groups[0]))} {self.put(_i32(groups[1]))}" if groups else "-1 - -"
        self.lines.append(f"paged_decode {layer} {slot} {g} {self.put(q)} {out}")
        self.after.append(lambda: check(self.get(out, np.float32, q.shape)))

    def fork(self, src, parent, add, held, dst, check):
        st = self.name()
        self.lines.append(f"pages_fork {src} {self.put(_i32(parent))} {self.put(_i32(add))} {self.put(_i32(held))} {dst} {st}")
        self.after.append(lambda: check(self.get(st, np.int32, 2)))

    def compact(self, src, held, dst, check):
        st = self.name()
        self.lines.append(f"pages_compact {src} {self.put(_i32(held))} {dst} {st}")
        self.after.append(lambda: check(self.get(st, np.int32, 2)))

    def done(self):
        with open(os.path.join(self.dir, "script.txt"), "w") as f:
            f.write("\n".join(self.lines + ["destroy", ""]))
        env = dict(os.environ, ASAN_OPTIONS="detect_stack_use_after_return=0", **self.env)
        r = subprocess.run([EMU_EXE, self.dir], capture_output=True, text=True, timeout=900, env=env)
        assert r.returncode == 0 and "attn_emu: ok" in r.stdout, r.stdout[-1500:] + r.stderr[-3000:]
        for f in self.after:
            f()
        return r.stdout


def _i32(a):
    return None if a is None else np.asarray(a, np.int32)


class GpuRunner(Runner):
    def __init__(self, **kw):
        super().__init__(**kw)
        self.G = g3attn()
        cfg = self.G.default_config(num_layers=self.layers, num_heads=self.hq, num_kv_heads=self.hkv, max_context=self.max_context,
                                    sliding_window=self.window)
        self.ctx = self.G.Context(cfg, self.max_context, self.tables[False].reshape(-1), self.tables[True].reshape(-1))
        self.keep, self.slots = [], {}

    def put(self, a):
        if a is None:
            return None
        b = DeviceBuffer.of(np.ascontiguousarray(a))
        self.keep.append(b)
        return b.ptr

    def buf(self, a):
        self.put(a)
        return self.keep[-1]

    def pool(self, p):
        self.p = p
        self.kb, self.vb = self.buf(p.pack(p.k)), self.buf(p.pack(p.v))
        self.pages = self.G.Pages(k=self.kb.ptr, v=self.vb.ptr, dtype=int(p.bf16), first_layer=p.first, num_layers=p.layers,
                                  num_pages=p.pages, page_size=p.ps, page_stride=p.page_stride, layer_stride=p.layer_stride)

    def seqs(self, slot, lens, table):
        n, t = self.buf(_i32(lens)), self.buf(_i32(table))
        s = self.G.Seqs(num_seqs=len(lens), kv_len=n.ptr, page_table=t.ptr, table_stride=table.shape[1])
        self.slots[slot] = (s, n, t)

    def pool_out(self, check):
        self.ctx.synchronize()
        dt = np.uint16 if self.p.bf16 else np.float32
        check(*(self.p.unpack(b.download(dt, self.p.size)) for b in (self.kb, self.vb)))

    def seqs_out(self, slot, shape, check):
        self.ctx.synchronize()
        s, n, t = self.slots[slot]
        check(n.download(np.int32, s.num_seqs), t.download(np.int32, shape))

    def batch(self, slot, n, q_start):
        return self.G.Batch(seqs=self.slots[slot][0], total_q=n, q_start=self.put(_i32(q_start)))

    def _out(self, q):
        return self.buf(np.full(q.shape, 4444.0, np.float32))

    def write(self, layer, slot, q_start, Q, K, V, qn, kn, check):
        out = self._out(Q)
        self.ctx.paged_write_device(layer, self.pages, self.batch(slot, len(Q), q_start), self.put(Q), self.put(K), self.put(V),
                                    self.put(qn), self.put(kn), out.ptr)
        self.ctx.synchronize()
        check(out.download(np.float32, Q.shape))

    def prefill(self, layer, slot, q_start, q, check):
        out = self._out(q)
        self.ctx.paged_prefill_device(layer, self.pages, self.batch(slot, len(q), q_start), self.put(q), out.ptr)
        self.ctx.synchronize()
        check(out.download(np.float32, q.shape))

    def decode(self, layer, slot, groups, q, check):
        out = self._out(q)
        g = self.G.Prefixes(num_groups=len(groups[1]), group_start=self.put(_i32(groups[0])), prefix_len=self.put(_i32(groups[1]))) if groups else None
        self.ctx.paged_decode_device(layer, self.pages, self.batch(slot, len(q), None), g, self.put(q), out.ptr)
        self.ctx.synchronize()
        check(out.download(np.float32, q.shape))

    def fork(self, src, parent, add, held, dst, check):
        st = self.buf(np.full(2, -5, np.int32))
        self.ctx.pages_fork_device(self.pages, self.slots[src][0], self.put(_i32(parent)), self.put(_i32(add)), self.put(_i32(held)),
                                   self.slots[dst][0], st.ptr)
        self.ctx.synchronize()
        check(st.download(np.int32, 2))

    def compact(self, src, held, dst, check):
        st = self.buf(np.full(2, -5, np.int32))
        self.ctx.pages_compact_device(self.pages, self.slots[src][0], self.put(_i32(held)), self.slots[dst][0], st.ptr)
        self.ctx.synchronize()
        check(st.download(np.int32, 2))

    def done(self):
        self.ctx.synchronize()
        for b in self.keep:
            b.free()
        self.ctx.close()
        return ""


# ------------------------------------------------------------------ whole cases

def run_prefill(r, layer, q_lens, lens, ps, bf16, seed=0, padding=0, bad=(), pool_kw=None, label="prefill", scale=2.0, kv_scale=1.0):
    """Packed prompts: q_lens new tokens of sequences of lens positions.
    padding: rows behind the last sequence; bad: (sequence, entry, page) table
    entries to spoil after the pool is filled."""
    rng = np.random.default_rng(seed)
    need = sum(-(-max(int(n), 0) // ps) for n in lens)
    pages = need + 2
    table = tables_for(rng, [max(n, 0) for n in lens], ps, pages)
    pool = Pool(rng, 1, pages, r.hkv, ps, bf16, first_layer=layer, **(pool_kw or {}))
    pool.fill(rng, table, lens, kv_scale)
    for b, j, page in bad:
        table[b, j] = page
    start = np.concatenate([[0], np.cumsum(q_lens)])
    n = int(start[-1])
    q = (rng.standard_normal((n + padding, r.hq, D)) * scale).astype(np.float32)
    r.pool(pool)
    r.seqs(0, lens, table)
    want = packed_attention(pool, layer, r.span(layer), table, lens, start, q[:n])

    def check(out):
        assert np.all(out[n:] == 4444.0), f"{label}: rows behind the last sequence were written"
        if n:
            check_close(out[:n], want, label)
    r.prefill(layer, 0, start, q, check)
    return want


def run_decode(r, layer, members, prefix, tail, ps, bf16, seed=0, groups=True, bad=(), label="decode", scale=2.0, pool_kw=None, lens=None):
    rng = np.random.default_rng(seed)
    group = [i for i, m in enumerate(members) for _ in range(m)]
    if lens is None:
        lens = [prefix[group[i]] + t for i, t in enumerate(tail)]
    first = np.concatenate([[0], np.cumsum(members)])
    shared = [(int(first[i]), m, prefix[i] // ps) for i, m in enumerate(members)]
    pages = sum(-(-n // ps) for n in lens) + 2
    table = tables_for(rng, lens, ps, pages, shared=shared)
    pool = Pool(rng, 1, pages, r.hkv, ps, bf16, first_layer=layer, **(pool_kw or {}))
    pool.fill(rng, table, lens)
    for i, m in enumerate(members):          # every member's copy of the prefix's last, partial page
        e, x = divmod(prefix[i], ps)
        for b in range(int(first[i]) + 1, int(first[i]) + m):
            if x:
                for a in (pool.k, pool.v):
                    a[:, table[b, e], :, :x] = a[:, table[first[i], e], :, :x]
    for b, j, page in bad:
        table[b, j] = page
    q = (rng.standard_normal((len(lens), r.hq, D)) * scale).astype(np.float32)
    r.pool(pool)
    r.seqs(0, lens, table)
    want = packed_attention(pool, layer, r.span(layer), table, lens, np.arange(len(lens) + 1), q)
    r.decode(layer, 0, (first, prefix) if groups else None, q, lambda out: check_close(out, want, label))
    return want


def run_write(r, layer, q_lens, lens, ps, bf16, norm=True, seed=0, padding=0, bad=(), pool_kw=None, label="write"):
    rng = np.random.default_rng(seed)
    pages = sum(-(-max(int(n), 0) // ps) for n in lens) + 2
    table = tables_for(rng, [max(n, 0) for n in lens], ps, pages)
    pool = Pool(rng, 2, pages, r.hkv, ps, bf16, first_layer=layer, fill=3.0, **(pool_kw or {}))
    for b, j, page in bad:
        table[b, j] = page
    start = np.concatenate([[0], np.cumsum(q_lens)])
    n = int(start[-1])
    Q, K, V = ((rng.standard_normal((n + padding, h, D)) * 3).astype(np.float32) for h in (r.hq, r.hkv, r.hkv))
    qn, kn = (to_bf16(rng.standard_normal(D) * 0.3) for _ in range(2)) if norm else (None, None)
    r.pool(pool)
    r.seqs(0, lens, table)
    wq, bq = np.full(Q.shape, 4444.0), np.zeros(Q.shape)
    wk, wv, bk = pool.k.astype(np.float64), pool.v.astype(np.float64), np.zeros(pool.k.shape)
    half = 2.0 ** -8 if bf16 else 0.0
    bv = np.zeros(pool.k.shape)
    for b in range(len(lens)):
        L = min(max(int(lens[b]), 0), table.shape[1] * ps)
        m = int(start[b + 1] - start[b])
        for i in range(m):
            t, pos = int(start[b]) + i, L - m + i
            if pos < 0 or pos >= r.max_context:
                continue
            wq[t], h = norm_rope(Q[t], qn, r.rope(layer), pos)
            bq[t] = 20 * 2.0 ** -24 * h
            page = table[b, pos // ps]
            if 0 <= page < pages:
                y, h = norm_rope(K[t], kn, r.rope(layer), pos)
                wk[0, page, :, pos % ps] = y
                bk[0, page, :, pos % ps] = half * np.abs(y) + 21 * 2.0 ** -24 * h
                wv[0, page, :, pos % ps] = V[t]
                bv[0, page, :, pos % ps] = half * np.abs(V[t])

    def near(got, want, bound, what):
        bad = np.abs(got - want) > bound
        assert not bad.any(), f"{label} {what}: {int(bad.sum())} off, worst {np.max(np.abs(got - want)):.2e}"
    r.write(layer, 0, start, Q, K, V, qn, kn, lambda out: near(out, wq, bq, "q"))
    r.pool_out(lambda k, v: (near(k, wk, bk, "k"), near(v, wv, bv, "v")))


def run_fork(r, lens, parent, add, ps, pages, bf16=False, held=None, seed=0, alias=False, stride=None, shared=(), layers=2, bad=(), label="fork",
             pool_kw=None, null=()):
    rng = np.random.default_rng(seed)
    free = [p for p in range(pages) if held is None or not held[p]]
    table = tables_for(rng, lens, ps, len(free), stride=stride, shared=shared)
    table = np.where(table >= 0, np.array(free, np.int32)[table], table).astype(np.int32)
    for b, j, page in bad:
        table[b, j] = page
    pool = Pool(rng, layers, pages, r.hkv, ps, bf16, **(pool_kw or {}))
    pool.k[...] = pool.round(rng.standard_normal(pool.k.shape))
    pool.v[...] = pool.round(rng.standard_normal(pool.v.shape))
    want_t, want_n, want_s, copies = fork(table, lens, parent, add, held, ps, pages)
    k, v = pool.k.copy(), pool.v.copy()
    for src, dst, n in copies:
        for a, o in ((k, pool.k), (v, pool.v)):
            a[:, dst, :, :n] = o[:, src, :, :n]
    r.pool(pool)
    r.seqs(0, lens, table)
    dst = 0 if alias else 1
    if not alias:
        r.seqs(1, np.full(len(parent), 99), np.full((len(parent), table.shape[1]), 99, np.int32))
    r.fork(0, None if "parent" in null else parent, None if "add" in null else add, held, dst,
           lambda st: _same(st, want_s, f"{label} status"))
    r.seqs_out(dst, want_t.shape, lambda n, t: (_same(n, want_n, f"{label} lengths"), _same(t, want_t, f"{label} tables")))
    r.pool_out(lambda a, b: (_same(a, k, f"{label} K"), _same(b, v, f"{label} V")))
    return want_t, want_n, want_s, copies


def run_compact(r, lens, ps, pages, bf16=False, held=None, seed=0, alias=False, shared=(), layers=2, label="compact", pool_kw=None, bad=()):
    rng = np.random.default_rng(seed)
    free = [p for p in range(pages) if held is None or not held[p]]
    table = tables_for(rng, lens, ps, len(free), shared=shared)
    table = np.where(table >= 0, np.array(free, np.int32)[table], table).astype(np.int32)
    for b, j, page in bad:
        table[b, j] = page
    pool = Pool(rng, layers, pages, r.hkv, ps, bf16, **(pool_kw or {}))
    pool.k[...] = pool.round(rng.standard_normal(pool.k.shape))
    pool.v[...] = pool.round(rng.standard_normal(pool.v.shape))
    want_t, want_n, want_s, moves = compact(table, lens, held, ps, pages)
    k, v = pool.k.copy(), pool.v.copy()
    for s, d in moves:
        k[:, d], v[:, d] = pool.k[:, s], pool.v[:, s]
    r.pool(pool)
    r.seqs(0, lens, table)
    dst = 0 if alias else 1
    if not alias:
        r.seqs(1, np.full(len(lens), 99), np.full(table.shape, 99, np.int32))
    r.compact(0, held, dst, lambda st: _same(st, want_s, f"{label} status"))
    r.seqs_out(dst, want_t.shape, lambda n, t: (_same(n, want_n, f"{label} lengths"), _same(t, want_t, f"{label} tables")))
    r.pool_out(lambda a, b: (_same(a, k, f"{label} K"), _same(b, v, f"{label} V")))
    return want_s


def _same(got, want, label):
    assert np.array_equal(np.asarray(got), np.asarray(want)), f"{label}: {got} is not {want}"


# ------------------------------------------------------------------ harder cases

def run_spoiled(r, layer, ps, bf16, spots, q_lens=None, lens=None, members=None, prefix=None, tail=None, seed=0, label="spoiled"):
    """Infinities and NaN in single elements of keys and values that some rows
    see: spots are (sequence, position, "k" or "v", value).  Rows that see one
    are NaN, all others as they are without."""
    rng = np.random.default_rng(seed)
    prompts = q_lens is not None
    if not prompts:
        group = [i for i, m in enumerate(members) for _ in range(m)]
        lens = [prefix[group[i]] + t for i, t in enumerate(tail)]
    first = np.concatenate([[0], np.cumsum(members if members else [len(lens)])])
    shared = [] if prompts else [(int(first[i]), m, prefix[i] // ps) for i, m in enumerate(members)]
    assert prompts or all(p % ps == 0 for p in prefix)      # a prefix is whole pages here
    table = tables_for(rng, lens, ps, sum(-(-n // ps) for n in lens) + 2, shared=shared)
    pool = Pool(rng, 1, int(table.max()) + 2, r.hkv, ps, bf16, first_layer=layer)
    pool.fill(rng, table, lens)
    start = np.concatenate([[0], np.cumsum(q_lens)]) if prompts else np.arange(len(lens) + 1)
    q = (rng.standard_normal((int(start[-1]), r.hq, D)) * 2).astype(np.float32)
    want = packed_attention(pool, layer, r.span(layer), table, lens, start, q)
    lost = np.zeros(want.shape[:2], bool)                   # [row][head]
    for i, (b, j, which, value) in enumerate(spots):
        h = i % r.hkv
        page = table[b, j // ps]
        getattr(pool, which)[0, page, h, j % ps, (37 * i + 5) % D] = value
        for s in range(len(lens)):
            if j // ps < table.shape[1] and table[s, j // ps] == page and j < lens[s]:
                n = start[s + 1] - start[s]
                for t in range(n):
                    pos = lens[s] - n + t
                    if j <= pos and j > pos - r.span(layer):
                        lost[start[s] + t, h * r.hq // r.hkv:(h + 1) * r.hq // r.hkv] = True
    assert lost.any() and not lost.all()

    def check(out):
        assert np.isnan(out[lost]).all(), f"{label}: a row that sees a spoiled key is not NaN"
        check_close(out[~lost], want[~lost], label)
    r.pool(pool)
    r.seqs(0, lens, table)
    if prompts:
        r.prefill(layer, 0, start, q, check)
    else:
        r.decode(layer, 0, (first, prefix), q, check)


SPOTS = [(0, 3, "v", np.nan), (0, 30, "k", np.inf), (0, 33, "v", -np.inf), (1, 40, "k", np.nan), (1, 61, "v", np.inf)]


def run_spoiled_all(r, layer, bf16):
    """Rows before a spoiled key, behind a window, in other heads and sequences."""
    run_spoiled(r, layer, 16, bf16, SPOTS, q_lens=[70, 25, 20], lens=[70, 77, 20], label="spoiled prompts")
    run_spoiled(r, layer, 16, bf16, [(0, 3, "v", np.nan), (0, 41, "k", -np.inf), (2, 70, "v", np.inf), (4, 1, "k", np.nan)],
                members=[3, 1, 1], prefix=[48, 0, 0], tail=[1, 9, 40, 30, 21], seed=1, label="spoiled members")


def run_faint(r, layer, bf16, keys=3000):
    """One key far ahead of the others, which are as much together: each
    probability is near 2^-12 of the largest and their sum is of its size.  The
    tolerance of check_close counts 22 bits of each probability, not of the
    largest one."""
    rng = np.random.default_rng(11)
    ps = 64
    table = tables_for(rng, [keys], ps, -(-keys // ps) + 1)
    pool = Pool(rng, 1, -(-keys // ps) + 1, r.hkv, ps, bf16, first_layer=layer, fill=0.0)
    k, v = np.zeros((keys, r.hkv, D)), np.zeros((keys, r.hkv, D))
    k[:, :, 0] = 1.0
    k[0, :, 0] = 1.0 + 16 * np.log(keys) / 64.0      # q . k / 16 rises by log(keys)
    v[...] = 1.0 + rng.standard_normal((1, 1, D)) / 4
    v[0] = rng.standard_normal((r.hkv, D))
    for p in range(keys):
        pool.k[0, table[0, p // ps], :, p % ps] = pool.round(k[p])
        pool.v[0, table[0, p // ps], :, p % ps] = pool.round(v[p])
    q = np.zeros((1, r.hq, D), np.float32)
    q[:, :, 0] = 64.0
    want = packed_attention(pool, layer, r.span(layer), table, [keys], [0, 1], q)
    r.pool(pool)
    r.seqs(0, [keys], table)
    r.prefill(layer, 0, [0, 1], q, lambda out: check_close(out, want, "faint keys, prefill"))
    r.decode(layer, 0, None, q, lambda out: check_close(out, want, "faint keys, decode"))


def run_serving(r, bf16, seed=0, rounds=4, ps=16):
    """The five calls as a server makes them, checked call by call against the
    oracles: prompts arrive, answers fork and grow, some end, the pool is
    compacted, a chunk follows."""
    rng = np.random.default_rng(seed)
    layers, pages = 2, 40
    pool = Pool(rng, layers, pages, r.hkv, ps, bf16, first_layer=4)       # layer 4 is local, 5 global
    width = 12
    lens, table = [0, 0, 0, 0], np.full((4, width), -1, np.int32)
    r.pool(pool)
    r.seqs(0, lens, table)
    half = 2.0 ** -8 if bf16 else 0.0
    qn, kn = to_bf16(rng.standard_normal(D) * 0.3), to_bf16(rng.standard_normal(D) * 0.3)

    def step(parent, add, slot, groups=None):
        """Fork, then per layer a write and the attention of the new tokens."""
        nonlocal table, lens
        parent, add = np.asarray(parent), np.asarray(add)
        want_t, want_n, want_s, copies = fork(table, lens, parent, add, None, ps, pages)
        assert want_s[1] == 0
        r.seqs(slot, np.full(len(parent), -7), np.full(want_t.shape, -7, np.int32))
        r.fork(1 - slot, parent, add, None, slot, lambda st: _same(st, want_s, "status"))
        r.seqs_out(slot, want_t.shape, lambda n, t: (_same(n, want_n, "lengths"), _same(t, want_t, "tables")))
        for src, dst, n in copies:
            for a in (pool.k, pool.v):
                a[:, dst, :, :n] = a[:, src, :, :n]
        table, lens = want_t, [int(n) for n in want_n]
        start = np.concatenate([[0], np.cumsum(add)])
        n = int(start[-1])
        for layer in (4, 5):
            Q, K, V = (rng.standard_normal((n, h, D)).astype(np.float32) for h in (r.hq, r.hkv, r.hkv))
            pos = np.concatenate([np.arange(lens[b] - add[b], lens[b]) for b in range(len(lens))])
            wq, bq = (np.stack(x) for x in zip(*(norm_rope(Q[t], qn, r.rope(layer), p) for t, p in enumerate(pos))))
            wk = np.stack([norm_rope(K[t], kn, r.rope(layer), p)[0] for t, p in enumerate(pos)])
            for t, p in enumerate(pos):
                b = int(np.searchsorted(start, t, "right")) - 1
                page = table[b, p // ps]
                pool.k[layer - 4, page, :, p % ps] = wk[t]
                pool.v[layer - 4, page, :, p % ps] = V[t]
            # what the attention reads is what was stored: off by the write's
            # rounding from these values, which a score feels through 256 terms
            # of either sign and an output directly
            rel = REL + 20 * 2.0 ** -24 * 4 + half
            want = packed_attention(pool, layer, r.span(layer), table, lens, start, wq.astype(np.float32))
            r.write(layer, slot, start, Q, K, V, qn, kn, lambda out, w=wq, b=bq: _near(out, w, 20 * 2.0 ** -24 * b, "q"))
            what = f"layer {layer} of {len(lens)} sequences"
            wq32 = wq.astype(np.float32)
            if np.all(add == 1):
                r.decode(layer, slot, groups, wq32, lambda out, w=want, m=what: check_close(out, w, "decode " + m, rel))
            else:
                r.prefill(layer, slot, start, wq32, lambda out, w=want, m=what: check_close(out, w, "prefill " + m, rel))

    def pack(slot):
        nonlocal table
        want_t, want_n, want_s, moves = compact(table, lens, None, ps, pages)
        r.compact(slot, None, slot, lambda st: _same(st, want_s, "compact status"))
        r.seqs_out(slot, want_t.shape, lambda n, t: (_same(n, want_n, "lengths"), _same(t, want_t, "tables")))
        old_k, old_v = pool.k.copy(), pool.v.copy()
        for s, d in moves:
            pool.k[:, d], pool.v[:, d] = old_k[:, s], old_v[:, s]
        table = want_t
        return len(moves)

    step([0, 1, 2], [37, 5, 50], 1)                          # three prompts
    step([0, 0, 0, 1, 2, 2], [1] * 6, 0, ([0, 3, 4, 6], [37, 5, 50]))   # and their first answers, six of them
    for i in range(rounds):
        step(range(6), [1] * 6, 1, ([0, 3, 4, 6], [37, 0, 50]))
        step(range(6), [1] * 6, 0, ([0, 3, 4, 6], [37, 0, 50]))
    step([1, 3, 5, -1], [0, 3, 20, 0], 1)                    # half of them end, others go on, an empty one
    assert pack(1) > 0
    step([0, 1, 2, 3], [1, 1, 1, 33], 0)                     # is the next prompt
    step([3, 0], [1, 1], 1)


def _near(got, want, bound, what):
    bad = np.abs(got - want) > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {np.max(np.abs(got - want)):.2e}"
