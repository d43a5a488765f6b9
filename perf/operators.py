"""What the paged-cache operators are measured on: page management of a K/V cache whose tables
live on the device (copy, fork, free, compact) and attention of a batch whose sequences share
a long prefix.

Shapes are those of this repository's two models (Stories110M: 12 heads of 64, no grouping,
fp16; Qwen3-0.6B: 16 query and 8 key/value heads of 128, bf16) and generic ones between them.

The cache.  A page holds 16 positions.  `pool` is [layers][pages][kv heads][K, V][16 * head_dim]
of 16-bit values; inside a K or V block the 8-value chunk c of row r sits at
(c / 8) * 1024 + r * 64 + ((c % 8) ^ (r % 8)) * 8.  `meta` packs the tables as 32-bit integers:
4 words (free pages, status, 0, 0), pages per slot, references per page, the free stack (the
next page to hand out is its last), and the block table [slots][pages per slot], -1 = none.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

#: False: the plain torch forms below; True: this repository's operators.
own = False

PAGE = 16
MAX_DRAW_BYTES = 1.0e9  # of a drawn case; the largest listed copy moves a little more
MAX_DRAW_FLOPS = 5e10   # of a drawn case; the largest listed attention does a little more


# ------------------------------------------------------------------------------- the cases
def listed():
    stories = {"dtype": "fp16", "heads": 12, "kv_heads": 12, "head_dim": 64}
    qwen3 = {"dtype": "bf16", "heads": 16, "kv_heads": 8, "head_dim": 128}
    return [
        # four samples of one short prompt, a few tokens in: the smallest decode call
        {"name": "attn_4_samples", "op": "attn", **stories, "layers": 2, "groups": 1, "members": 4, "prefix": 112,
         "suffix": 24, "rows": 1, "idle": False, "lse": False},
        # a full batch in eight families, each on its own system prompt, at unequal progress
        {"name": "attn_8_families_of_32", "op": "attn", **qwen3, "layers": 1, "groups": 8, "members": 32,
         "prefix": 2048, "suffix": 1024, "rows": 1, "idle": True, "lse": True},
        # 64 answers over one long document
        {"name": "attn_64_on_32k", "op": "attn", **qwen3, "layers": 1, "groups": 1, "members": 64, "prefix": 32768,
         "suffix": 192, "rows": 1, "idle": False, "lse": False},
        # user prompts of unequal length after a common system prompt, in one prefill call
        {"name": "attn_24_prompts", "op": "attn", **qwen3, "layers": 1, "groups": 1, "members": 24, "prefix": 2048,
         "suffix": 203, "rows": 203, "idle": False, "lse": False},
        # three pages of one sequence of the small model; a quarter of a pool of the large one
        {"name": "copy_3_pages", "op": "copy", **stories, "layers": 12, "pages": 96, "count": 3},
        {"name": "copy_2048_pages", "op": "copy", **qwen3, "layers": 4, "pages": 8192, "count": 2048},
        # four samples leave one prompt; 64 beams of unequal length fan out eightfold
        {"name": "fork_1_into_4", "op": "fork", **stories, "layers": 12, "pages": 96, "families": 1, "fan": 4,
         "length": 100, "room": 16},
        {"name": "fork_64_into_512", "op": "fork", **qwen3, "layers": 4, "pages": 8192, "families": 64, "fan": 8,
         "length": 1100, "room": 40},
        # one sequence ends; half of a large batch of short sequences over long shared prompts ends
        {"name": "free_1_of_8", "op": "free", **stories, "layers": 1, "pages": 256, "families": 2, "fan": 4,
         "length": 200, "room": 0, "count": 1},
        {"name": "free_512_of_1024", "op": "free", **stories, "layers": 1, "pages": 16384, "families": 32, "fan": 32,
         "length": 2040, "room": 150, "count": 512},
        # a small pool after a few requests; a large one with half of its pages live, anywhere
        {"name": "compact_96", "op": "compact", **stories, "layers": 12, "pages": 96, "families": 2, "fan": 3,
         "length": 130, "room": 40},
        {"name": "compact_8192", "op": "compact", **qwen3, "layers": 4, "pages": 8192, "families": 96, "fan": 4,
         "length": 600, "room": 80},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kv, hd = rng.choice([(12, 64), (8, 128), (1, 64), (2, 128), (3, 64), (4, 128), (6, 128), (5, 64)])
        case = {"op": rng.choice(["attn", "attn", "attn", "copy", "fork", "free", "compact"]),
                "dtype": rng.choice(["fp16", "bf16"]), "heads": kv * rng.choice([1, 1, 2, 3, 4, 7, 8]), "kv_heads": kv,
                "head_dim": hd, "layers": rng.choice([1, 2, 3])}
        if case["op"] == "attn":
            case |= {"groups": _log(rng, 1, 12), "members": _log(rng, 1, 96), "prefix": PAGE * _log(rng, 1, 2048),
                     "suffix": _log(rng, 1, 1100), "rows": 1, "idle": rng.random() < 0.5, "lse": rng.random() < 0.5}
            if rng.random() < 0.3:
                case["rows"] = _log(rng, 2, 200)
                case["suffix"] = max(case["suffix"], case["rows"])
            seqs = case["groups"] * case["members"]
            plain = 4.0 * seqs * case["rows"] * case["heads"] * (case["prefix"] + case["suffix"])  # scores in f32
            plain += 8.0 * seqs * case["suffix"] * kv * hd
            if plain > 6e9:
                continue
        elif case["op"] == "copy":
            case |= {"pages": _log(rng, 16, 8192)}
            case["count"] = _log(rng, 1, max(1, case["pages"] // 2))
        else:
            case |= {"families": _log(rng, 1, 64), "fan": _log(rng, 1, 32), "length": _log(rng, 1, 2048),
                     "room": _log(rng, 1, 160)}
            if case["op"] == "free":
                case["count"] = _log(rng, 1, case["families"] * case["fan"])
            used = case["families"] * (-(-case["length"] // PAGE) + case["fan"] * (-(-case["room"] // PAGE) + 2))
            case["pages"] = used + 24 + _log(rng, 16, 2 * used + 16)
        if "pages" in case and case["layers"] * case["pages"] * kv * hd * 64 > 3e9:
            continue
        w = work(case)
        if w["bytes"] <= MAX_DRAW_BYTES and w["flops"] <= MAX_DRAW_FLOPS:
            return case


# ------------------------------------------------------------------------------- the inputs
def _dtype(case):
    return {"fp16": torch.float16, "bf16": torch.bfloat16}[case["dtype"]]


def _attn_lengths(case, seed):
    """Per family its prefix; per sequence its query rows and the positions it sees."""
    r = np.random.RandomState(seed % (1 << 31))
    G, M = case["groups"], case["members"]
    prefix = case["prefix"] - PAGE * r.randint(0, case["prefix"] // PAGE // 2 + 1, G) if G > 1 else np.array([case["prefix"]])
    prefix = np.maximum(prefix, PAGE)
    rows = np.random.RandomState(G * M).randint(case["rows"] // 4 + 1, case["rows"] + 1, G * M)  # of every seed: the shapes
    if case["rows"] == 1:
        rows[:] = 1
    ctx = np.repeat(prefix, M) + np.maximum(rows, r.randint(1, case["suffix"] + 1, G * M))
    if case["idle"]:
        ctx[r.randint(0, G * M)] = 0  # an idle place of a fixed batch: it sees nothing
    return prefix.astype(np.int64), rows.astype(np.int64), ctx.astype(np.int64)


def _families(case, seed):
    """The tables of a pool with families of sequences that share their prompt's full pages."""
    r = np.random.RandomState(seed % (1 << 31))
    F, fan, n = case["families"], case["fan"], case["pages"]
    slots = F * fan if case["op"] != "fork" else F * (1 + fan) + 2 * F
    most = -(-(case["length"] + case["room"]) // PAGE) + 2
    table = np.full((slots, most), -1, np.int64)
    npages = np.zeros(slots, np.int64)
    ids = r.permutation(n)
    at = 0
    lengths = np.maximum(1, r.randint(case["length"] // 2, case["length"] + 1, F))
    for f in range(F):
        held = -(-lengths[f] // PAGE)
        table_f, at = ids[at:at + held], at + held
        if case["op"] == "fork":  # one sequence to fork; its children's slots are still empty
            table[f, :held], npages[f] = table_f, held
            continue
        for s in range(f * fan, (f + 1) * fan):
            keep = held if s == f * fan else lengths[f] // PAGE
            more = int(r.randint(0, -(-case["room"] // PAGE) + 1)) + held - keep
            table[s, :keep] = table_f[:keep]
            table[s, keep:keep + more] = ids[at:at + more]
            at += more
            npages[s] = keep + more
    assert at <= n, "the case's pool is too small"
    held = table[table >= 0]
    refs = np.bincount(held, minlength=n)
    free = np.full(n, -1, np.int64)
    empty = r.permutation(np.flatnonzero(refs == 0))
    free[:empty.size] = empty
    meta = np.concatenate([[empty.size, 0, 0, 0], npages, refs, free, table.reshape(-1)]).astype(np.int32)
    return meta, slots, most, lengths, r


def _pool(case, pages, g):
    shape = (case["layers"], pages, case["kv_heads"], 2, PAGE * case["head_dim"])
    pool = torch.empty(shape, dtype=_dtype(case), device="cuda")
    return pool.normal_(generator=g)


def _split(meta, case_slots, most, n):
    """Views of a packed table: (words, pages per slot, references, free stack, block table)."""
    a, b, c = 4 + case_slots, 4 + case_slots + n, 4 + case_slots + 2 * n
    return meta[:4], meta[4:a], meta[a:b], meta[b:c], meta[c:].view(case_slots, most)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = lambda a, t=torch.int32: torch.as_tensor(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    st = {"case": case}
    if case["op"] == "attn":
        prefix, rows, ctx = _attn_lengths(case, seed)
        G, M = case["groups"], case["members"]
        n_seqs, most = G * M, int(-(-(case["prefix"] + max(case["suffix"], case["rows"])) // PAGE))
        r = np.random.RandomState((seed + 1) % (1 << 31))
        own_pages = np.maximum(0, -(-ctx // PAGE) - np.repeat(prefix // PAGE, M))
        n_pages = int(own_pages.sum() + (prefix // PAGE).sum()) + 5
        ids = r.permutation(n_pages)
        table = np.full((n_seqs, most), -1, np.int64)
        at = 0
        for f in range(G):
            shared = prefix[f] // PAGE
            table[f * M:(f + 1) * M, :shared] = ids[at:at + shared]
            at += shared
            for s in range(f * M, (f + 1) * M):
                table[s, shared:shared + own_pages[s]] = ids[at:at + own_pages[s]]
                at += own_pages[s]
        npages = (table >= 0).sum(1)
        refs = np.bincount(table[table >= 0], minlength=n_pages)
        free = np.full(n_pages, -1, np.int64)
        free[:5] = ids[at:at + 5]
        st["meta"] = dev(np.concatenate([[5, 0, 0, 0], npages, refs, free, table.reshape(-1)]))
        st["pool"] = _pool(case, n_pages, g)
        n_rows = int(rows.sum())
        st["q"] = torch.empty((n_rows, case["heads"], case["head_dim"]), dtype=_dtype(case), device="cuda").normal_(generator=g)
        st["ctx"] = dev(ctx)
        st["layer"] = case["layers"] - 1
        st["shape"] = (n_seqs, most, n_pages)
        # the batch's layout, kept while its sequences run: padded indexes for the plain form
        start = np.concatenate([[0], np.cumsum(rows)])
        R = int(rows.max())
        at_row = start[:-1, None] + np.arange(R)[None]
        st["row_of"] = dev(np.where(np.arange(R)[None] < rows[:, None], at_row, n_rows), torch.int64)
        st["place"] = dev(np.repeat(np.arange(n_seqs), rows) * R + np.concatenate([np.arange(k) for k in rows]), torch.int64)
        st["rows"], st["prefix"] = dev(rows), dev(prefix)
        st["most"] = (int(prefix.max()), int(max(1, (-(-ctx // PAGE) - np.repeat(prefix // PAGE, M)).max()) * PAGE))
        st["layout"] = ([M] * G, prefix.tolist(), rows.tolist())
        return st
    if case["op"] == "copy":
        r = np.random.RandomState(seed % (1 << 31))
        n, k = case["pages"], case["count"]
        ids = r.permutation(n)
        st["pool"] = _pool(case, n, g)
        st["src"], st["dst"] = dev(ids[:k]), dev(ids[n - k:])
        meta, slots, most = np.zeros(4 + 1 + 2 * n + 1, np.int32), 1, 1  # its tables play no part
    else:
        meta, slots, most, lengths, r = _families(case, seed)
        st["pool"] = _pool(case, case["pages"], g)
    if case["op"] == "fork":
        F, fan = case["families"], case["fan"]
        # each family's children, then one new sequence and one that grows in place
        parents = np.concatenate([np.repeat(np.arange(F), fan), [-1], [0]])
        lens = np.concatenate([np.repeat(lengths, fan) - r.randint(0, 2, F * fan) * (np.repeat(lengths, fan) // 2), [0], [0]])
        rooms = lens + r.randint(1, case["room"] + 1, lens.size)
        rooms[-1] = lengths[0] + case["room"]
        children = np.concatenate([F + r.permutation(F * fan + 1), [0]])
        order = r.permutation(parents.size)
        st |= {"parents": dev(parents[order]), "children": dev(children[order]), "lens": dev(lens[order]), "rooms": dev(rooms[order])}
    if case["op"] == "free":
        st["slots"] = dev(r.permutation(slots)[:case["count"]])
    st["before"] = dev(meta)
    st["meta"] = st["before"].clone()
    st["shape"] = (slots, most, case["pages"])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:  # the handles that a program keeps: the cache over these buffers, and its batch's plan
        package = str(Path(__file__).resolve().parent.parent / "ane-training-experiments_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from ane.paged import PagedCache, PrefixPlan
        slots, most, n = st["shape"]
        st["cache"] = PagedCache(case["dtype"], case["layers"], n, case["kv_heads"], case["head_dim"], slots, most,
                                 pool=st["pool"], meta=st["meta"])
        if case["op"] == "attn":
            sizes, prefix, rows = st["layout"]
            st["plan"] = PrefixPlan(st["cache"], case["heads"], range(slots), rows, sizes, prefix, max_ctx=most * PAGE)
    return st


# ------------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if case["op"] == "attn":
        if not own:
            return _plain_attn(st)
        lse = torch.empty(st["q"].shape[:2], dtype=torch.float32, device="cuda") if case["lse"] else None
        out = st["plan"].attend(st["layer"], st["q"], st["ctx"], lse=lse)
        return {"out": out, "lse": lse} if case["lse"] else {"out": out}
    if case["op"] == "copy":
        if own:
            st["cache"].copy(st["src"], st["dst"])
        else:
            st["pool"][:, st["dst"].long()] = st["pool"][:, st["src"].long()]
        return {"pool": st["pool"]}
    # the tables as this step finds them: the call before changed them
    st["meta"].copy_(st["before"])
    if case["op"] == "fork":
        if own:
            st["cache"].fork(st["parents"], st["children"], st["lens"], st["rooms"])
        else:
            _plain_fork(st)
        return {"meta": st["meta"], "pool": st["pool"]}
    if case["op"] == "free":
        if own:
            st["cache"].free(st["slots"])
        else:
            _plain_free(st)
        return {"meta": st["meta"]}
    if own:
        st["cache"].compact()
    else:
        _plain_compact(st)
    return {"meta": st["meta"], "pool": st["pool"]}


def _plain_fork(st):
    slots, most, n = st["shape"]
    words, npages, refs, free, table = _split(st["meta"], slots, most, n)
    parent, child = st["parents"].long(), st["children"].long()
    grow = parent == child
    held = torch.where(parent >= 0, npages[parent.clamp(min=0)], 0).long()
    keep = torch.where(grow, held, st["lens"].long() // PAGE)
    part = ~grow & (st["lens"] % PAGE > 0)
    new = ((st["rooms"].long() + PAGE - 1) // PAGE - keep).clamp(min=0)
    off = torch.cumsum(new, 0) - new
    j = torch.arange(most, device="cuda")[None]
    old = table[parent.clamp(min=0)]
    shared = (j < keep[:, None]) & ~grow[:, None]
    fresh = (j >= keep[:, None]) & (j < (keep + new)[:, None])
    page = free[(words[0].long() - 1 - off[:, None] - (j - keep[:, None])).clamp(0, n - 1)]
    src = old.gather(1, keep.clamp(max=most - 1)[:, None])[:, 0][part].long()
    dst = page.gather(1, keep.clamp(max=most - 1)[:, None])[:, 0][part].long()
    table[child] = torch.where(shared, old, torch.where(fresh, page, table[child]))
    refs.index_add_(0, old[shared].long(), torch.ones((), dtype=torch.int32, device="cuda").expand(int(shared.sum())))
    refs[page[fresh].long()] = 1
    npages[child] = (keep + new).int()
    words[0] -= new.sum().int()
    st["pool"][:, dst] = st["pool"][:, src]


def _plain_free(st):
    slots, most, n = st["shape"]
    words, npages, refs, free, table = _split(st["meta"], slots, most, n)
    gone = st["slots"].long()
    rows = table[gone]
    ids = rows[torch.arange(most, device="cuda")[None] < npages[gone][:, None]].long()
    before = refs.clone()
    refs.index_add_(0, ids, torch.full_like(ids, -1, dtype=torch.int32))
    empty = torch.nonzero((refs == 0) & (before > 0))[:, 0]
    free[words[0].long() + torch.arange(empty.numel(), device="cuda")] = empty.int()
    words[0] += empty.numel()
    table[gone] = -1
    npages[gone] = 0


def _plain_compact(st):
    slots, most, n = st["shape"]
    words, npages, refs, free, table = _split(st["meta"], slots, most, n)
    ids = torch.arange(n, device="cuda")
    live = refs > 0
    count = live.sum()
    src = torch.nonzero(live & (ids >= count))[:, 0]
    dst = torch.nonzero(~live & (ids < count))[:, 0]
    to = ids.int()
    to[src] = dst.int()
    st["pool"][:, dst] = st["pool"][:, src]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    empty = n - count
    free.copy_(torch.where(ids < empty, (n - 1 - ids).int(), free))
    words[0] = empty.int()


def _swizzle(hd):
    r, d = torch.meshgrid(torch.arange(PAGE, device="cuda"), torch.arange(hd, device="cuda"), indexing="ij")
    c = d // 8
    return ((c // 8) * 1024 + r * 64 + ((c % 8) ^ (r % 8)) * 8 + d % 8).reshape(-1)


def _plain_attn(st):
    case = st["case"]
    slots, most, n = st["shape"]
    _, _, _, _, table = _split(st["meta"], slots, most, n)
    G, M, H, KV, hd = case["groups"], case["members"], case["heads"], case["kv_heads"], case["head_dim"]
    S, gq = G * M, H // KV
    P, X = st["most"]
    at = _swizzle(hd)

    def pages(ids):  # [a, p] page numbers -> K, V [a, kv, 16 p, hd] in 32 bits
        got = st["pool"][st["layer"]][ids.clamp(min=0).long()].float().index_select(-1, at)
        got = got.view(*ids.shape, KV, 2, PAGE, hd).permute(3, 0, 2, 1, 4, 5).reshape(2, ids.shape[0], KV, -1, hd)
        return got[0], got[1]

    q = torch.cat([st["q"].float(), torch.zeros(1, H, hd, device="cuda")])[st["row_of"]]  # [S, R, H, hd]
    R = q.shape[1]
    q = q.view(S, R, KV, gq, hd).permute(0, 2, 1, 3, 4).reshape(S, KV, R * gq, hd) / math.sqrt(hd)
    i = torch.arange(R, device="cuda").repeat_interleave(gq)
    pos = (st["ctx"] - st["rows"])[:, None] + i[None]  # [S, R * gq]
    prefix = st["prefix"].repeat_interleave(M)  # [S]

    k, v = pages(table[::M, : P // PAGE])
    by_group = lambda x: x.view(G, M, KV, R * gq, -1).transpose(1, 2).reshape(G, KV, M * R * gq, -1)  # noqa: E731
    by_seq = lambda x: x.view(G, KV, M, R * gq, -1).transpose(1, 2).reshape(S, KV, R * gq, -1)  # noqa: E731
    s0 = by_seq(by_group(q) @ k.transpose(-1, -2))
    t = torch.arange(P, device="cuda")
    s0.masked_fill_(~((t < prefix[:, None, None]) & (t <= pos[:, :, None]))[:, None], -math.inf)

    t = torch.arange(X, device="cuda")
    entry = (prefix // PAGE)[:, None] + torch.arange(X // PAGE, device="cuda")[None]
    k1, v1 = pages(table.gather(1, entry.clamp(max=most - 1).long()))
    v1 = v1.masked_fill(((prefix[:, None] + t) >= st["ctx"][:, None])[:, None, :, None], 0.0)
    s1 = q @ k1.transpose(-1, -2)
    s1.masked_fill_(~((prefix[:, None, None] + t) <= pos[:, :, None])[:, None], -math.inf)

    m = torch.maximum(s0.amax(-1, keepdim=True), s1.amax(-1, keepdim=True))
    top = torch.where(torch.isinf(m), 0.0, m)
    p0, p1 = torch.exp(s0 - top), torch.exp(s1 - top)
    l = p0.sum(-1, keepdim=True) + p1.sum(-1, keepdim=True)
    o = by_seq(by_group(p0) @ v) + p1 @ v1
    o = torch.where(l > 0, o / torch.where(l > 0, l, 1.0), 0.0)
    flat = lambda x: x.view(S, KV, R, gq, -1).transpose(1, 2).reshape(S * R, H, -1)[st["place"]]  # noqa: E731
    out = {"out": flat(o).to(_dtype(case))}
    if case["lse"]:
        out["lse"] = flat(top + torch.log(l))[..., 0].contiguous()
    return out


# ------------------------------------------------------------------------------- what it cannot do without
def _expected(case):
    """Mean figures of a case with families: pages that a prompt holds, new pages of a sequence."""
    return 0.75 * case["length"] / PAGE + 0.5, 0.5 * case["room"] / PAGE + 0.5


def work(case):
    page = case["layers"] * case["kv_heads"] * 2 * PAGE * case["head_dim"] * 2  # bytes of a page in every layer
    if case["op"] == "attn":
        prefix, rows, ctx = _attn_lengths(case, 1)
        own_positions = np.maximum(0, ctx - np.repeat(prefix, case["members"])).sum()
        kv = 2 * 2 * case["kv_heads"] * case["head_dim"]
        row = case["heads"] * case["head_dim"] * 2
        seen = (rows * np.maximum(0, ctx - (rows - 1) / 2.0)).sum()
        n = rows.sum()
        return {"bytes": float((prefix.sum() + own_positions) * kv + 2 * n * row + (4 * n * case["heads"] if case["lse"] else 0)
                               + 4 * ((prefix // PAGE).sum() + own_positions / PAGE)),
                "flops": float(4.0 * case["heads"] * case["head_dim"] * seen)}
    if case["op"] == "copy":
        return {"bytes": float(case["count"] * (2 * page + 8)), "flops": 0.0}
    held, new = _expected(case)
    n, seqs = case["pages"], case["families"] * case.get("fan", 1)
    if case["op"] == "fork":  # half of the children keep the whole prompt, half of them half of it
        return {"bytes": float(seqs * (15 / 16 * 2 * page + 0.75 * held * 16 + new * 12 + 24)), "flops": 0.0}
    if case["op"] == "free":  # entries read and cleared, references changed, emptied pages pushed
        return {"bytes": float(case["count"] * ((held + new) * 16 + 12) + 16), "flops": 0.0}
    live = case["families"] * (held + case["fan"] * new)
    moved = live * (1 - min(1.0, live / n))  # references read and written, entries read, the free stack written
    return {"bytes": float(moved * 2 * page + 8 * n + 4 * (n - live) + seqs * (held + new) * 4), "flops": 0.0}


# ------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, seed, st)
    pool = st["pool"].double()
    if case["op"] == "copy":
        for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
            pool[:, b] = st["pool"][:, a].double()
        return {"pool": pool}
    slots, most, n = st["shape"]
    words, npages, refs, free, table = (x.cpu().numpy().copy() for x in _split(st["before"], slots, most, n))
    moves = []
    if case["op"] == "fork":
        left = int(words[0])
        was = npages.copy()
        for p, c, length, room in zip(*(st[k].tolist() for k in ("parents", "children", "lens", "rooms"))):
            have = int(was[p]) if p == c else length // PAGE
            if p != c:
                for j in range(have):
                    table[c, j] = table[p, j]
                    refs[table[p, j]] += 1
            count = have
            while count * PAGE < room:
                left -= 1
                table[c, count] = free[left]
                refs[free[left]] = 1
                count += 1
            if p != c and length % PAGE:
                moves.append((int(table[p, have]), int(table[c, have])))
            npages[c] = count
        words[0] = left
    elif case["op"] == "free":
        empty = []
        for s in st["slots"].tolist():
            for j in range(int(npages[s])):
                refs[table[s, j]] -= 1
                if refs[table[s, j]] == 0:
                    empty.append(int(table[s, j]))
            npages[s] = 0
            table[s] = -1
        for p in sorted(empty):
            free[words[0]] = p
            words[0] += 1
    else:
        count = int((refs > 0).sum())
        holes = iter([p for p in range(count) if refs[p] == 0])
        for p in range(count, n):
            if refs[p] > 0:
                h = next(holes)
                moves.append((p, h))
                refs[h], refs[p] = refs[p], 0
        to = dict(moves)
        for s in range(slots):
            for j in range(int(npages[s])):
                table[s, j] = to.get(int(table[s, j]), int(table[s, j]))
        for k in range(n - count):
            free[k] = n - 1 - k
        words[0] = n - count
    meta = torch.as_tensor(np.concatenate([words, npages, refs, free, table.reshape(-1)])).to("cuda", torch.int32)
    if case["op"] == "free":
        return {"meta": meta}
    for a, b in moves:
        pool[:, b] = st["pool"][:, a].double()
    return {"meta": meta, "pool": pool}


def _exact_attn(case, seed, st):
    prefix, rows, ctx = _attn_lengths(case, seed)
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if 4.0 * H * hd * float((rows * ctx).sum()) > 3e12:
        return None
    slots, most, n = st["shape"]
    table = st["meta"][-slots * most:].view(slots, most).cpu().numpy()
    layer = st["pool"][st["layer"]]
    spot = np.zeros((PAGE, hd), np.int64)
    for r in range(PAGE):
        for d in range(hd):
            spot[r, d] = (d // 64) * 1024 + r * 64 + (((d // 8) % 8) ^ (r % 8)) * 8 + d % 8
    spot = torch.as_tensor(spot.reshape(-1), device="cuda")
    outs, lses, at = [], [], 0
    for s in range(slots):
        q = st["q"][at:at + int(rows[s])].double()
        at += int(rows[s])
        L = int(ctx[s])
        if L == 0:
            outs.append(torch.zeros_like(q))
            lses.append(torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda"))
            continue
        ids = torch.as_tensor(table[s, : -(-L // PAGE)].astype(np.int64), device="cuda")
        kv = layer[ids].double()[..., spot].view(-1, KV, 2, PAGE, hd)
        k = kv[:, :, 0].transpose(0, 1).reshape(KV, -1, hd)[:, :L].repeat_interleave(H // KV, 0)
        v = kv[:, :, 1].transpose(0, 1).reshape(KV, -1, hd)[:, :L].repeat_interleave(H // KV, 0)
        score = torch.einsum("rhd,htd->hrt", q, k) * hd ** -0.5
        for r in range(q.shape[0]):
            score[:, r, L - q.shape[0] + r + 1:] = -math.inf
        lse = torch.logsumexp(score, -1)
        outs.append(torch.einsum("hrt,htd->rhd", torch.exp(score - lse[..., None]), v))
        lses.append(lse.transpose(0, 1))
    got = {"out": torch.cat(outs)}
    if case["lse"]:
        got["lse"] = torch.cat(lses)
    return got
