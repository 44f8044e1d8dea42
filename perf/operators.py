"""The operators of a KV cache in pages, as cases that can be timed and checked:
writing the tokens of many sequences, attention of packed prompts, attention of
one token a sequence with prefixes that several sequences share, and forking and
compacting the sequences themselves.

`own = False` computes them in plain torch operations, `own = True` calls the
entry points of include/g3attn.h as gemma3.c_amd/g3attn.py binds them, on the
context's stream.

Layouts: a pool of pages per matrix [layer][page][KV head][row][256], fp32 or
bf16; a page table [sequence][entry] (entry j holds positions j * page size ..,
-1 where there is none) and a length for each sequence; packed rows of several
sequences [row][head][256] with the offset of each sequence's first row.
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 256          # head_dim
WINDOW = 1024    # sliding window of the local layers
EPS = 1e-6
THETA = {"local": 1e4, "global": 1e6}
LAYER = {"local": 0, "global": 5}   # a layer of each kind in the model's pattern


# ------------------------------------------------------------------ cases

def _join(v):
    return ",".join(str(int(x)) for x in v)


def _split(s):
    return [int(x) for x in s.split(",")] if s else []


def _spread(rng, n, lo, hi):
    """n lengths between lo and hi, even over their logarithm."""
    return [_log(rng, lo, hi) for _ in range(n)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def listed():
    r = random.Random(11)
    return [
        # 48 conversations, each one token further: latency more than bytes
        dict(name="write_step_48", kind="write", layer="local", dtype="f32", hq=8, hkv=4, ps=16, norm=True,
             q=_join([1] * 48), hist=_join(_spread(r, 48, 20, 4000))),
        # five prompts of a batch that arrive together
        dict(name="write_prompts_8192", kind="write", layer="global", dtype="bf16", hq=8, hkv=4, ps=32, norm=True,
             q="4000,2500,1000,500,192", hist="0,0,700,33,0"),
        # short prompts through a local layer: few tiles, latency
        dict(name="prefill_short_9", kind="prefill", layer="local", dtype="f32", hq=8, hkv=4, ps=16,
             q="120,77,64,33,17,5,90,1,49", hist="0,0,0,0,0,0,0,0,0"),
        # prompts of a document service, packed, through a global layer
        dict(name="prefill_packed_8192", kind="prefill", layer="global", dtype="f32", hq=8, hkv=4, ps=16,
             q="5000,1800,900,492", hist="0,0,0,0"),
        # follow-up messages over cached histories, half the bytes a key
        dict(name="prefill_chunks_bf16", kind="prefill", layer="global", dtype="bf16", hq=16, hkv=8, ps=64,
             q="512,333,257,700,129", hist="3000,6000,1111,0,9000"),
        # answers sampled from one long prompt
        dict(name="decode_shared_64", kind="decode", layer="global", dtype="f32", hq=8, hkv=4, ps=16,
             members="64", prefix="8192", tail=_join(_spread(r, 64, 1, 600))),
        # three system prompts, conversations of different lengths behind them
        dict(name="decode_groups_bf16", kind="decode", layer="global", dtype="bf16", hq=16, hkv=8, ps=32,
             members="20,7,21", prefix="2000,5001,333", tail=_join(_spread(r, 48, 10, 2000))),
        # unrelated conversations: nothing shared
        dict(name="decode_ragged_8", kind="decode", layer="global", dtype="f32", hq=8, hkv=4, ps=16,
             members=_join([1] * 8), prefix=_join([0] * 8), tail="37,4000,1203,650,2222,91,3100,511"),
        # one step of a beam search: beams fork, grow by a token, the others end
        dict(name="fork_beam_16", kind="fork", dtype="f32", hkv=4, ps=16, layers=6, pages=2048, parents=16, children=16,
             len_lo=100, len_hi=900, add=1, shape=3),
        # many samples from each prompt's end, over every layer
        dict(name="fork_samples_256", kind="fork", dtype="bf16", hkv=4, ps=64, layers=34, pages=1024, parents=32,
             children=256, len_lo=300, len_hi=1500, add=1, shape=5),
        # a small pool after a few sequences have ended
        dict(name="compact_small", kind="compact", dtype="f32", hkv=4, ps=16, layers=6, pages=512, seqs=7, len_lo=200,
             len_hi=800, shape=7),
        # a large pool, fragmented by a day's traffic
        dict(name="compact_large", kind="compact", dtype="bf16", hkv=4, ps=32, layers=34, pages=2500, seqs=40, len_lo=300,
             len_hi=2500, shape=9),
    ]


def draw(rng):
    kind = rng.choice(["write", "prefill", "prefill", "decode", "decode", "fork", "compact"])
    dtype = rng.choice(["f32", "bf16"])
    hq, hkv = rng.choice([(8, 4), (8, 4), (16, 8), (4, 1), (4, 4)])
    ps = rng.choice([16, 32, 64, 128])
    layer = rng.choice(["local", "global"])
    if kind == "write":
        if rng.random() < 0.4:
            n = _log(rng, 1, 300)
            q, hist = [1] * n, _spread(rng, n, 1, 12000)
        else:
            n = rng.randint(1, 9)
            q, hist = _spread(rng, n, 1, 1500), [rng.choice([0, _log(rng, 1, 4000)]) for _ in range(n)]
        return dict(kind=kind, layer=layer, dtype=dtype, hq=hq, hkv=hkv, ps=ps, norm=rng.random() < 0.8, q=_join(q), hist=_join(hist))
    if kind == "prefill":
        n = _log(rng, 1, 12)
        most = _log(rng, 10, 6000 if hq <= 8 else 3500) // n + 1
        q = [rng.choice([most, _log(rng, 1, most)]) for _ in range(n)]
        hist = [rng.choice([0, 0, _log(rng, 1, 8000 // n)]) for _ in range(n)]
        return dict(kind=kind, layer=layer, dtype=dtype, hq=hq, hkv=hkv, ps=ps, q=_join(q), hist=_join(hist))
    if kind == "decode":
        g = rng.choice([0, 1, 1, 2, 4])
        if g == 0:
            n = _log(rng, 1, 40)
            return dict(kind=kind, layer=layer, dtype=dtype, hq=hq, hkv=hkv, ps=ps, members=_join([1] * n), prefix=_join([0] * n),
                        tail=_join(_spread(rng, n, 1, 8000)))
        members = _spread(rng, g, 1, 64 // g)
        return dict(kind=kind, layer=layer, dtype=dtype, hq=hq, hkv=hkv, ps=ps, members=_join(members),
                    prefix=_join(_spread(rng, g, 20, 7000)), tail=_join(_spread(rng, sum(members), 1, 1000)))
    layers = rng.choice([1, 6, 12])
    if kind == "fork":
        parents = _log(rng, 1, 60)
        hi = _log(rng, 20, 1500)
        pages = parents * (hi // ps + 2) + 512
        return dict(kind=kind, dtype=dtype, hkv=hkv, ps=ps, layers=layers, pages=pages, parents=parents, children=_log(rng, 1, 200),
                    len_lo=max(1, hi // 6), len_hi=hi, add=rng.choice([0, 1, 1, 7, 100]), shape=rng.randrange(1 << 20))
    seqs = _log(rng, 1, 40)
    hi = _log(rng, 20, 2500)
    return dict(kind=kind, dtype=dtype, hkv=hkv, ps=ps, layers=layers, pages=seqs * (hi // ps + 2) + rng.randint(10, 300), seqs=seqs,
                len_lo=max(1, hi // 6), len_hi=hi, shape=rng.randrange(1 << 20))


# ------------------------------------------------------------------ inputs

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 31)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


_tables = {}


def _rope(which, max_context):
    """RoPE table [max_context][D / 2][cos, sin] in fp32, angles in 64 bits."""
    key = (which, max_context)
    if key not in _tables:
        if len(_tables) > 3:
            _tables.clear()
        freq = THETA[which] ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2 / D)
        angle = torch.arange(max_context, dtype=torch.float64, device="cuda")[:, None] * freq[None]
        _tables[key] = torch.stack([angle.cos(), angle.sin()], -1).float()
    return _tables[key]


def _page_tables(g, lens, ps, shared=None, spare=0):
    """Tables over randomly ordered pages; `shared` = [(members, pages)]: groups
    of sequences whose first entries are the same pages."""
    need = [-(-n // ps) for n in lens]
    common = [0] * len(lens)
    lead = list(range(len(lens)))
    if shared:
        i = 0
        for members, pages in shared:
            for j in range(members):
                common[i + j], lead[i + j] = (pages, i)
            i += members
    total = sum(n if lead[i] == i else n - min(n, common[i]) for i, n in enumerate(need)) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    table = np.full((len(lens), max(need) + 1), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        c = 0 if lead[i] == i else min(n, common[i])
        table[i, :c] = table[lead[i], :c]
        table[i, c:n] = order[at:at + n - c]
        at += n - c
    return torch.from_numpy(table).cuda(), total


def _gain(g):
    return torch.randn(D, generator=g, device="cuda", dtype=torch.bfloat16).mul_(1 / 8)


def _prepare_packed(case, seed):
    """write and prefill: packed rows of sequences with a history."""
    g = _gen(seed)
    q, hist = _split(case["q"]), _split(case["hist"])
    lens = [a + b for a, b in zip(q, hist)]
    table, pages = _page_tables(g, lens, case["ps"], spare=3)
    dt = TORCH[case["dtype"]]
    n = sum(q)
    s = dict(case=case, table=table, lens=_int(lens), start=_int([0] + list(np.cumsum(q))))
    s["max_context"] = 1 << max(13, (max(lens) - 1).bit_length())
    # cached keys have been through the norm: about one a dim
    s["k"] = _randn(g, pages, case["hkv"], case["ps"], D, dtype=dt)
    s["v"] = _randn(g, pages, case["hkv"], case["ps"], D, dtype=dt)
    if case["kind"] == "write":
        s["Q"], s["K"], s["V"] = (_randn(g, n, h, D, scale=1.7) for h in (case["hq"], case["hkv"], case["hkv"]))
        s["qn"], s["kn"] = (_gain(g), _gain(g)) if case["norm"] else (None, None)
        s["rope"] = _rope(case["layer"], s["max_context"])
        s["out"] = torch.zeros(n, case["hq"], D, device="cuda")
    else:
        # the norms' gains make scores a few units wide
        s["q"] = _randn(g, n, case["hq"], D, scale=2.0)
        s["out"] = torch.zeros(n, case["hq"], D, device="cuda")
    return s


def _decode_shape(case):
    members, prefix, tail = _split(case["members"]), _split(case["prefix"]), _split(case["tail"])
    group = [i for i, m in enumerate(members) for _ in range(m)]
    return members, prefix, [prefix[group[i]] + t for i, t in enumerate(tail)]


def _prepare_decode(case, seed):
    g = _gen(seed)
    members, prefix, lens = _decode_shape(case)
    # a fork shares the prefix's full pages; each sequence has its own copy of the last, partial one
    table, pages = _page_tables(g, lens, case["ps"], [(m, p // case["ps"]) for m, p in zip(members, prefix)], spare=3)
    dt = TORCH[case["dtype"]]
    s = dict(case=case, table=table, lens=_int(lens), group=_int([0] + list(np.cumsum(members))), prefix=_int(prefix))
    s["max_context"] = 1 << max(13, (max(lens) - 1).bit_length())
    s["k"] = _randn(g, pages, case["hkv"], case["ps"], D, dtype=dt)
    s["v"] = _randn(g, pages, case["hkv"], case["ps"], D, dtype=dt)
    first = 0
    for m, p in zip(members, prefix):
        if p % case["ps"] and m > 1:
            e, r = p // case["ps"], p % case["ps"]
            src, dst = table[first, e].long(), table[first + 1:first + m, e].long()
            for x in (s["k"], s["v"]):
                x[dst, :, :r] = x[src, :, :r]
        first += m
    s["q"] = _randn(g, len(lens), case["hq"], D, scale=2.0)
    s["out"] = torch.zeros(len(lens), case["hq"], D, device="cuda")
    return s


def _fork_shape(case):
    """Lengths of the parents, and each child's parent and growth."""
    r = random.Random(case["shape"])
    lens = _spread(r, case["parents"], case["len_lo"], case["len_hi"])
    parent = [r.randrange(case["parents"]) for _ in range(case["children"])]
    if case["children"] > 2:
        parent[r.randrange(case["children"])] = -1      # a slot that falls empty
    return lens, parent, [case["add"]] * case["children"]


def _prepare_pages(case, seed):
    g = _gen(seed)
    r = random.Random(case["shape"])
    if case["kind"] == "fork":
        lens, parent, add = _fork_shape(case)
    else:
        lens = _spread(r, case["seqs"], case["len_lo"], case["len_hi"])
    table, used = _page_tables(g, lens, case["ps"])
    grown = (max(lens) + case.get("add", 0)) // case["ps"] + 2
    wide = torch.full((len(lens), grown), -1, dtype=torch.int32, device="cuda")
    # the pages in use lie anywhere in the pool
    place = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
    w = min(grown, table.shape[1])
    t = table[:, :w]
    wide[:, :w] = torch.where(t >= 0, place[t.clamp_min(0).long()], t)
    dt = TORCH[case["dtype"]]
    shape = (case["layers"], case["pages"], case["hkv"], case["ps"], D)
    s = dict(case=case, table=wide, lens=_int(lens), k=_randn(g, *shape, dtype=dt), v=_randn(g, *shape, dtype=dt))
    rows = case["children"] if case["kind"] == "fork" else len(lens)
    if case["kind"] == "fork":
        s["parent"], s["add"] = _int(parent), _int(add)
    s["table_out"] = torch.zeros(rows, grown, dtype=torch.int32, device="cuda")
    s["lens_out"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s["status"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    kind = case["kind"]
    return (_prepare_packed if kind in ("write", "prefill") else _prepare_decode if kind == "decode" else _prepare_pages)(case, seed)


# ------------------------------------------------------------------ the framework's calls

_contexts = {}


def _binding():
    if "g3attn" not in sys.modules:
        spec = importlib.util.spec_from_file_location("g3attn", os.path.join(os.getcwd(), "gemma3.c_amd", "g3attn.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["g3attn"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["g3attn"]


def _context(hq, hkv, max_context):
    """The engine's context; it has one, and every call goes through it."""
    key = (hq, hkv, max_context)
    if key not in _contexts:
        _contexts.clear()
        G = _binding()
        cfg = G.default_config(num_layers=6, num_heads=hq, num_kv_heads=hkv, max_context=max_context, sliding_window=WINDOW, rmsnorm_eps=EPS)
        tables = [_rope(w, max_context).cpu().numpy().reshape(-1) for w in ("local", "global")]
        _contexts[key] = G.Context(cfg, max_context, *tables)
    return _contexts[key]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(s):
    """One call of the entry point, with the descriptors that the program keeps."""
    case, G = s["case"], _binding()
    kind = case["kind"]
    ctx = _context(case.get("hq", case["hkv"]), case["hkv"], s.get("max_context", 8192))
    if "pages" not in s:
        dtype = G.PAGE_F32 if case["dtype"] == "f32" else G.PAGE_BF16
        k = s["k"]
        one = k.dim() == 4
        # a pool of one of the model's layers, or of all from the first
        s["pages"] = G.Pages(k=k.data_ptr(), v=s["v"].data_ptr(), dtype=dtype, first_layer=LAYER[case["layer"]] if one else 0,
                             num_layers=1 if one else k.shape[0], num_pages=k.shape[-4], page_size=case["ps"],
                             page_stride=k.stride(-4), layer_stride=0 if one else k.stride(0))
        seqs = dict(num_seqs=len(s["lens"]), kv_len=s["lens"].data_ptr(), page_table=s["table"].data_ptr(), table_stride=s["table"].shape[1])
        if kind in ("fork", "compact"):
            s["in"] = G.Seqs(**seqs)
            s["to"] = G.Seqs(num_seqs=len(s["lens_out"]), kv_len=s["lens_out"].data_ptr(), page_table=s["table_out"].data_ptr(),
                             table_stride=s["table_out"].shape[1])
        else:
            s["in"] = G.Batch(seqs=G.Seqs(**seqs), total_q=len(s["out"]), q_start=None if kind == "decode" else s["start"].data_ptr())
            if kind == "decode":
                s["groups"] = G.Prefixes(num_groups=len(s["prefix"]), group_start=s["group"].data_ptr(), prefix_len=s["prefix"].data_ptr())
    if kind == "write":
        ctx.paged_write_device(LAYER[case["layer"]], s["pages"], s["in"], s["Q"].data_ptr(), s["K"].data_ptr(), s["V"].data_ptr(),
                               _ptr(s["qn"]), _ptr(s["kn"]), s["out"].data_ptr())
    elif kind == "prefill":
        ctx.paged_prefill_device(LAYER[case["layer"]], s["pages"], s["in"], s["q"].data_ptr(), s["out"].data_ptr())
    elif kind == "decode":
        ctx.paged_decode_device(LAYER[case["layer"]], s["pages"], s["in"], s["groups"], s["q"].data_ptr(), s["out"].data_ptr())
    elif kind == "fork":
        ctx.pages_fork_device(s["pages"], s["in"], s["parent"].data_ptr(), s["add"].data_ptr(), None, s["to"], s["status"].data_ptr())
    else:
        ctx.pages_compact_device(s["pages"], s["in"], None, s["to"], s["status"].data_ptr())


# ------------------------------------------------------------------ the plain forms

def _places(s, ps):
    """Of every packed row: its sequence, position, page and row in the page."""
    q = (s["start"][1:] - s["start"][:-1]).long()
    n = len(s["out"])
    seq = torch.repeat_interleave(torch.arange(len(q), device="cuda"), q, output_size=n)
    pos = torch.arange(n, device="cuda") - s["start"].long()[seq] + (s["lens"].long() - q)[seq]
    return seq, pos, s["table"][seq, pos // ps].long(), pos % ps


def _norm_rotate(x, w, rope, pos):
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w.to(x.dtype))
    c, n = rope[pos].to(x.dtype).unbind(-1)
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, n = c[:, None], n[:, None]
    return torch.cat([a * c - b * n, a * n + b * c], -1)


def _plain_write(s):
    _, pos, page, row = _places(s, s["case"]["ps"])
    s["out"].copy_(_norm_rotate(s["Q"], s["qn"], s["rope"], pos))
    s["k"][page, :, row] = _norm_rotate(s["K"], s["kn"], s["rope"], pos).to(s["k"].dtype)
    s["v"][page, :, row] = s["V"].to(s["v"].dtype)


def _gather(pages, table, n):
    """Rows 0 .. n - 1 of every sequence [sequence][KV head][n][D], in fp32."""
    ps = pages.shape[2]
    t = table[:, :-(-n // ps)].clamp_min(0).long()
    x = pages[t].float()                                  # [seq][entry][head][row][D]
    return x.permute(0, 2, 1, 3, 4).reshape(len(t), pages.shape[1], -1, D)[:, :, :n].contiguous()


def _attend(q, k, v, seen):
    """q [B][Hkv][rows][D], k / v [B][Hkv][n][D], seen [B][1][rows][n] -> [B][Hkv][rows][D]."""
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(D)
    score.masked_fill_(~seen, -math.inf)
    score -= score.amax(-1, keepdim=True).clamp_min(-3e38)
    score.exp_()
    return torch.matmul(score, v) / score.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_prefill(s):
    """Every sequence padded to the longest."""
    case = s["case"]
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    q = [int(x) for x in _split(case["q"])]
    most, longest, B = max(q), max(a + b for a, b in zip(q, _split(case["hist"]))), len(q)
    seq, pos, _, _ = _places(s, case["ps"])
    at = torch.arange(len(seq), device="cuda") - s["start"].long()[seq]
    rows = torch.zeros(B, most, case["hq"], D, device="cuda")
    rows[seq, at] = s["q"]
    where = torch.full((B, most), -1, dtype=torch.long, device="cuda")
    where[seq, at] = pos
    rows = rows.reshape(B, most, hkv, group, D).permute(0, 2, 1, 3, 4).reshape(B, hkv, most * group, D)
    j = torch.arange(longest, device="cuda")
    i = where.repeat_interleave(group, 1)[:, None, :, None]
    seen = (j <= i) & (j > i - (WINDOW if case["layer"] == "local" else 1 << 40))
    o = _attend(rows.contiguous(), _gather(s["k"], s["table"], longest), _gather(s["v"], s["table"], longest), seen)
    o = o.reshape(B, hkv, most, group, D).permute(0, 2, 1, 3, 4).reshape(B, most, case["hq"], D)
    s["out"].copy_(o[seq, at])


def _plain_decode(s):
    """Every sequence with its own copy of its prefix."""
    case = s["case"]
    hkv, B = case["hkv"], len(s["lens"])
    longest = max(_decode_shape(case)[2])
    j = torch.arange(longest, device="cuda")
    n = s["lens"].long()[:, None, None, None]
    seen = (j < n) & (j >= n - (WINDOW if case["layer"] == "local" else 1 << 40))
    o = _attend(s["q"].reshape(B, hkv, -1, D), _gather(s["k"], s["table"], longest), _gather(s["v"], s["table"], longest), seen)
    s["out"].copy_(o.reshape(B, case["hq"], D))


def _in_use(table, n, ps, pages):
    """How many sequences hold each page, from tables whose first ceil(n / ps) entries count."""
    held = torch.arange(table.shape[1], device="cuda")[None] < ((n + ps - 1) // ps)[:, None]
    return torch.bincount(table[held].long(), minlength=pages), held


def _plain_fork(s):
    ps, pages, width = s["case"]["ps"], s["k"].shape[1], s["table"].shape[1]
    p = s["parent"].long()
    b = torch.arange(len(p), device="cuda")
    real = (p >= 0) & (p < len(s["lens"]))
    row = s["table"][p.clamp(0, len(s["lens"]) - 1)]
    old = torch.where(real, s["lens"].long()[p.clamp(0, len(s["lens"]) - 1)], 0).clamp(0, width * ps)
    want = torch.where(real, old + s["add"].long(), 0).clamp_min(0)
    fits = want <= width * ps
    want = torch.where(fits, want, old)
    keep = torch.minimum(old, want)
    kept, full = (keep + ps - 1) // ps, (want + ps - 1) // ps
    ref, _ = _in_use(row, keep, ps, pages)
    tail = row.gather(1, (old // ps).clamp_max(width - 1)[:, None])[:, 0].long()
    writes = (want > old) & (old % ps != 0)
    tail = torch.where(writes, tail, 0)
    writers = torch.zeros(pages, dtype=torch.long, device="cuda").index_add_(0, tail, writes.long())
    first = torch.full((pages,), 1 << 30, dtype=torch.long, device="cuda")
    first.scatter_reduce_(0, tail, torch.where(writes, b, 1 << 30), "amin")
    apart = writes & ~((first[tail] == b) & (writers[tail] == ref[tail]))
    need = full - kept + apart.long()
    free = torch.argsort((ref > 0).to(torch.int8), stable=True)
    offset = torch.cumsum(need, 0) - need
    granted = fits & ((need == 0) | (offset + need <= (ref == 0).sum()))
    after = torch.where(granted, want, old)
    apart = apart & granted
    full = torch.where(granted, full, kept)
    j = torch.arange(width, device="cuda")[None]
    fresh = free[(offset[:, None] + (j - kept[:, None]) + apart.long()[:, None]).clamp(0, pages - 1)].int()
    table = torch.where(j < kept[:, None], row, torch.where(j < full[:, None], fresh, -1))
    copy = torch.where(apart, free[offset.clamp(0, pages - 1)], 0)
    table = torch.where(apart[:, None] & (j == (old // ps)[:, None]), copy[:, None].int(), table)
    s["table_out"].copy_(table)
    s["lens_out"].copy_(after)
    used = (ref > 0).sum() + torch.where(granted, need, 0).sum()
    s["status"].copy_(torch.stack([used, (~granted).sum()]))
    src, dst, rows = tail[apart], copy[apart], (old % ps)[apart]
    mine = (torch.arange(ps, device="cuda")[None] < rows[:, None])[None, :, None, :, None]
    s["k"][:, dst] = torch.where(mine, s["k"][:, src], s["k"][:, dst])
    s["v"][:, dst] = torch.where(mine, s["v"][:, src], s["v"][:, dst])


def _plain_compact(s):
    ps, pages = s["case"]["ps"], s["k"].shape[1]
    n = s["lens"].long()
    ref, held = _in_use(s["table"], n, ps, pages)
    used = (ref > 0).sum()
    at = torch.arange(pages, device="cuda")
    src = at[(ref > 0) & (at >= used)]
    dst = at[(ref == 0) & (at < used)]
    now = at.clone()
    now[src] = dst
    s["table_out"].copy_(torch.where(held, now[s["table"].clamp_min(0).long()].int(), -1))
    s["lens_out"].copy_(n)
    s["status"].copy_(torch.stack([used, torch.full_like(used, len(src))]))
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]


_plain = {"write": _plain_write, "prefill": _plain_prefill, "decode": _plain_decode, "fork": _plain_fork, "compact": _plain_compact}


def run(s):
    kind = s["case"]["kind"]
    if own:
        _call(s)
    else:
        _plain[kind](s)
    if kind == "write":
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if kind in ("prefill", "decode"):
        return s["out"]
    return {"table": s["table_out"], "len": s["lens_out"], "status": s["status"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------ work

def _bytes(case):
    return 4 if case["dtype"] == "f32" else 2


def _copied(case):
    """Rows (fork) or pages (compact) that have to be copied, by the definition.
    A compaction's pages in use lie at random places: what is expected of it."""
    ps = case["ps"]
    if case["kind"] == "compact":
        r = random.Random(case["shape"])
        used = sum(-(-n // ps) for n in _spread(r, case["seqs"], case["len_lo"], case["len_hi"]))
        return used * (case["pages"] - used) // case["pages"] * ps
    lens, parent, add = _fork_shape(case)
    seen, rows = set(), 0
    for p, a in zip(parent, add):
        if p < 0 or a <= 0 or lens[p] % ps == 0:
            continue
        rows += lens[p] % ps if p in seen else 0
        seen.add(p)
    return rows


def work(case):
    kind, e = case["kind"], _bytes(case)
    if kind in ("fork", "compact"):
        rows = _copied(case)
        tables = 8 * (case.get("parents", case.get("seqs")) + case.get("children", case.get("seqs"))) * (case["len_hi"] // case["ps"] + 1)
        return dict(bytes=rows * case["layers"] * 2 * case["hkv"] * D * e * 2 + tables, flops=0)
    hq, hkv = case["hq"], case["hkv"]
    W = WINDOW if case["layer"] == "local" else 1 << 40
    if kind == "write":
        n = sum(_split(case["q"]))
        return dict(bytes=n * D * (8 * hq + (4 + e) * 2 * hkv + 4), flops=n * D * 10 * (hq + hkv))
    if kind == "prefill":
        pairs = rows = n = 0
        for q, h in zip(_split(case["q"]), _split(case["hist"])):
            full = max(0, min(q, W - h))     # tokens whose window reaches position 0
            pairs += full * h + full * (full + 1) // 2 + (q - full) * W
            rows += q + min(h, W - 1)
            n += q
        return dict(bytes=n * hq * D * 8 + rows * 2 * hkv * D * e, flops=4 * D * hq * pairs)
    members, prefix, lens = _decode_shape(case)
    pairs = sum(min(n, W) for n in lens)
    first = rows = 0
    for m, p in zip(members, prefix):
        part = lens[first:first + m]
        rows += sum(min(W, n - p) for n in part) + max(0, p - min(max(0, n - W) for n in part))
        first += m
    return dict(bytes=len(lens) * hq * D * 8 + rows * 2 * hkv * D * e, flops=4 * D * hq * pairs)


# ------------------------------------------------------------------ 64 bits

def _exact_rows(pages, table, n):
    ps = pages.shape[2]
    return torch.cat([pages[int(t)].double() for t in table[:-(-n // ps)]], 1)[:, :n]      # [head][n][D]


def _exact_attention(case, s):
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    W = WINDOW if case["layer"] == "local" else 1 << 40
    lens, table = s["lens"].tolist(), s["table"].cpu()
    q = _split(case["q"]) if case["kind"] == "prefill" else [1] * len(lens)
    out = torch.zeros(sum(q), case["hq"], D, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, m) in enumerate(zip(lens, q)):
        lo = max(0, n - m + 1 - W)
        k, v = (_exact_rows(s[x], table[b], n)[:, lo:] for x in "kv")
        for i in range(0, m, 1024):
            e = min(m, i + 1024)
            pos = torch.arange(n - m + i, n - m + e, device="cuda")[:, None]
            j = torch.arange(lo, n, device="cuda")[None]
            unseen = (j > pos) | (j <= pos - W)
            for h in range(case["hq"]):
                x = s["q"][first + i:first + e, h].double() @ k[h // group].T / math.sqrt(D)
                out[first + i:first + e, h] = torch.softmax(x.masked_fill(unseen, -math.inf), -1) @ v[h // group]
        first += m
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "compact"):
        return None            # whole numbers, and rows that are moved
    s = prepare(case, seed)
    if kind in ("prefill", "decode"):
        return _exact_attention(case, s)
    q, hist, ps = _split(case["q"]), _split(case["hist"]), case["ps"]
    pos = torch.cat([torch.arange(h, h + n) for n, h in zip(q, hist)]).cuda()
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(q)]).cuda()
    page = s["table"][seq, pos // ps].long()
    t = s["rope"][pos].double()[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS) * (1 + w.double())
        z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * torch.complex(t[..., 0], t[..., 1])
        return torch.cat([z.real, z.imag], -1)

    k, v = s["k"].double(), s["v"].double()
    k[page, :, pos % ps] = turned(s["K"], s["kn"])
    v[page, :, pos % ps] = s["V"].double()
    return {"q": turned(s["Q"], s["qn"]), "k": k, "v": v}
