"""The measured workloads of search over the paged cache: what a decode loop with beams or drafted
tokens asks of this library between two steps of the model.

  tree      attention of drafted tokens (a tree per sequence, or one token each) over the cached
            history of several sequences and the drafted tokens' own K and V rows
  path      the accepted tokens' K and V rows of every layer into the pages of their sequences
  fork      the sequences of the next step from those of the last one: shared pages, a copy of the
            last page where two would write into it
  compact   the pages in use moved to the front of the arenas
  beam      the best continuations of each request's beams over the vocabulary

Sizes of heads, layers and vocabulary are those of the models in this repository's configurations and
bench, or generic. A case fixes how much there is to do; the seed only which pages, parents and values.
"""
import math

import torch

own = False

F32, F16, Q8_0 = 0, 1, 8
TYPES = {"F32": F32, "F16": F16, "Q8_0": Q8_0}
BLOCK = 16  # tokens per page
DEV = "cuda"


def _tree(name, cache, seqs, tokens, past_min, past_max, heads, kv_heads, head_dim, ragged=False):
    return {"name": name, "op": "tree", "cache": cache, "seqs": seqs, "tokens": tokens, "past_min": past_min,
            "past_max": past_max, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "ragged": ragged}


def _path(name, cache, seqs, tokens, accepted, past, layers, kv_heads, head_dim):
    return {"name": name, "op": "path", "cache": cache, "seqs": seqs, "tokens": tokens, "accepted": accepted,
            "past": past, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim}


def _fork(name, cache, batch, beams, survivors, prefix, layers, kv_heads, head_dim):
    return {"name": name, "op": "fork", "cache": cache, "batch": batch, "beams": beams, "survivors": survivors,
            "prefix": prefix, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim}


def _compact(name, cache, pages, live, moved, layers, kv_heads, head_dim):
    return {"name": name, "op": "compact", "cache": cache, "pages": pages, "live": live, "moved": moved,
            "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim}


def _beam(name, dtype, batch, beams, vocab, n_out):
    return {"name": name, "op": "beam", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab, "n_out": n_out}


def listed():
    return [
        # one user's small drafted tree over a short chat: launch latency
        _tree("tree_one_f16", "F16", 1, 7, 100, 100, 16, 8, 128),
        # a served batch with drafted trees of up to 24 tokens, sequences of different lengths
        _tree("tree_batch_f16", "F16", 8, 24, 1500, 4096, 32, 8, 128, ragged=True),
        # one long document, a full tree of 64 tokens
        _tree("tree_long_q8_0", "Q8_0", 1, 64, 32768, 32768, 32, 8, 128),
        # the next token of every beam of a batch, one KV head, fp32 cache
        _tree("beams_decode_f32", "F32", 37, 1, 301, 1501, 8, 1, 256),
        # one user's accepted tokens into a 28-layer cache: latency
        _path("path_one_f16", "F16", 1, 7, 3, 100, 28, 8, 128),
        # a batch's accepted tokens into a 36-layer fp32 cache
        _path("path_batch_f32", "F32", 16, 24, 5, 500, 36, 8, 128),
        # one request's four beams go on from three of them: latency, one page copied
        _fork("fork_one_f16", "F16", 1, 4, 3, 9, 28, 8, 128),
        # sixteen requests' eight beams, five of each go on
        _fork("fork_batch_f16", "F16", 16, 8, 5, 14, 36, 8, 128),
        # a small arena with a few holes
        _compact("compact_small_f16", "F16", 120, 70, 11, 16, 8, 64),
        # a cache that half of its requests have left
        _compact("compact_half_f32", "F32", 501, 250, 117, 36, 8, 64),
        # one request's beams over a large vocabulary
        _beam("beam_one_f32", "F32", 1, 4, 151936, 8),
        # a batch of 32 requests with eight beams each
        _beam("beam_batch_f32", "F32", 32, 8, 151936, 16),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "path", "fork", "compact", "beam", "beam"])
    head_dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8]) if head_dim < 256 else rng.choice([1, 2, 4])
    cache = rng.choice(["F16", "F32"])
    layers = rng.choice([1, 5, 16, 28, 36])
    if op == "tree":
        while True:
            tokens = rng.choice([1, 1, _log_uniform(rng, 1, 100)])
            past_max = rng.choice([0, 5]) if rng.random() < 0.1 else _log_uniform(rng, 1, 32768)
            past_min = past_max if rng.random() < 0.3 else rng.randint(0, past_max)
            case = _tree("", rng.choice(["F16", "Q8_0", "F32"]), _log_uniform(rng, 1, 40), tokens, past_min,
                         past_max, kv_heads * rng.choice([1, 2, 3, 4, 7, 8]), kv_heads, head_dim,
                         ragged=rng.random() < 0.5)
            w = work(case)
            if w["flops"] <= 3.5e10 and w["bytes"] <= 2.5e8:
                break
    elif op == "path":
        tokens = _log_uniform(rng, 1, 64)
        case = _path("", cache, _log_uniform(rng, 1, 16), tokens, rng.randint(1, min(tokens, 8)), rng.randint(0, 600),
                     layers, kv_heads, head_dim)
    elif op == "fork":
        beams = rng.randint(1, 8)
        case = _fork("", cache, _log_uniform(rng, 1, 12), beams, rng.randint(1, beams), rng.randint(0, 14), layers,
                     min(kv_heads, 4), min(head_dim, 128))
    elif op == "compact":
        pages = _log_uniform(rng, 8, 500)
        live = rng.randint(1, pages - 1)
        case = _compact("", cache, pages, live, rng.randint(0, min(live, pages - live)), min(layers, 28), min(kv_heads, 4),
                        min(head_dim, 128))
    else:
        beams = rng.randint(1, 8)
        case = _beam("", rng.choice(["F32", "F16"]), _log_uniform(rng, 1, 24), beams, _log_uniform(rng, 50, 151936),
                     rng.randint(1, 2 * beams))
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs
def _row_bytes(cache, elems):
    return {"F32": 4 * elems, "F16": 2 * elems, "Q8_0": elems // 32 * 34}[cache]


def _arena(cache, pages, layers, elems, gen):
    """Bytes of an arena of `pages` pages, its values normal."""
    n = pages * layers * BLOCK * elems
    if cache == "Q8_0":
        raw = torch.empty((n // 32, 34), dtype=torch.uint8, device=DEV)
        d = (0.5 + torch.rand((n // 32, 1), generator=gen, device=DEV)) / 60.0
        raw[:, :2] = d.half().view(torch.uint8)
        raw[:, 2:] = torch.clamp(torch.randn((n // 32, 32), generator=gen, device=DEV) * 50.0, -127, 127).round().to(
            torch.int8).view(torch.uint8)
        return raw.view(-1)
    dtype = torch.float16 if cache == "F16" else torch.float32
    return torch.randn(n, generator=gen, device=DEV).to(dtype).view(torch.uint8)


def _pasts(case):
    """The sequences' histories, spread evenly over the case's range (the seed only orders them)."""
    n, lo, hi = case["seqs"], case["past_min"], case["past_max"]
    return [hi - (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _drafts(case):
    n, t = case["seqs"], case["tokens"]
    return [t - (i * t // (2 * n) if case["ragged"] else 0) for i in range(n)]


def _cache(case, pages, layers, k, v):
    """The program's cache over the arenas (only where the framework's own calls are made)."""
    import densecore_amd as dc
    c = dc.PagedKVCache(TYPES[case["cache"]], 1, layers, case["kv_heads"], case["head_dim"], device=DEV)
    c.n_blocks, c.k, c.v = pages, k, v
    return c


def _prepare_tree(case, seed, gen, rng):
    s, t, h, g, d = (case[x] for x in ("seqs", "tokens", "heads", "kv_heads", "head_dim"))
    past = torch.tensor(_pasts(case))[torch.randperm(s, generator=rng)]
    width = max((case["past_max"] + BLOCK - 1) // BLOCK, 1)
    used = (past + BLOCK - 1) // BLOCK
    pages = int(used.sum()) + 3
    order, tables, at = torch.randperm(pages, generator=rng), torch.full((s, width), -1), 0
    for i in range(s):
        n = int(used[i])
        tables[i, :n] = order[at:at + n]
        at += n
    drafts = torch.tensor(_drafts(case))
    words = (t + 63) // 64
    seen = torch.zeros((s, t, t), dtype=torch.bool)
    for i in range(s):
        for j in range(t):  # a random tree: the parent of a drafted token is an earlier one, or the history
            p = int(torch.randint(-1, j, (1,), generator=rng)) if j else -1
            if p >= 0:
                seen[i, j] = seen[i, p]
            seen[i, j, j] = True
    bits = torch.zeros((s, t, words), dtype=torch.int64)
    for w in range(words):
        for b in range(min(64, t - 64 * w)):
            one = 1 << b if b < 63 else -(1 << 63)
            bits[:, :, w] |= torch.where(seen[:, :, 64 * w + b], one, 0)
    st = {"layers": 2, "layer": 1, "pages": pages, "k": _arena(case["cache"], pages, 2, g * d, gen),
          "v": _arena(case["cache"], pages, 2, g * d, gen), "tables": tables.int().to(DEV),
          "past": past.int().to(DEV), "drafts": drafts.int().to(DEV), "mask": bits.to(DEV),
          "q": torch.randn((s * t, h * d), generator=gen, device=DEV) * 2.0,
          "kc": torch.randn((s * t, g * d), generator=gen, device=DEV),
          "vc": torch.randn((s * t, g * d), generator=gen, device=DEV),
          "scale": 1.0 / math.sqrt(d), "host_past": past.tolist(), "host_drafts": drafts.tolist()}
    if own:
        import densecore_amd as dc
        st["cache_obj"] = _cache(case, pages, 2, st["k"], st["v"])
        st["out"] = torch.empty((s * t, h * d), device=DEV)
        need = dc.kv_tree_attention_workspace_size(h, g, d, s, t, case["past_max"])
        st["ws"] = torch.empty(max(need, 256), dtype=torch.uint8, device=DEV)
    return st


def _prepare_path(case, seed, gen, rng):
    s, t, n, layers = case["seqs"], case["tokens"], case["accepted"], case["layers"]
    elems = case["kv_heads"] * case["head_dim"]
    past = [max(case["past"] - 37 * i, 0) for i in range(s)]
    width = (case["past"] + n + BLOCK - 1) // BLOCK
    # the pages that the accepted tokens fall into, and no others of the history
    need = [sorted({(p + j) // BLOCK for j in range(n)}) for p in past]
    pages = sum(len(b) for b in need) + 2
    order, tables, at = torch.randperm(pages, generator=rng), torch.full((s, width), -1), 0
    for i, blocks in enumerate(need):
        for b in blocks:
            tables[i, b] = order[at]
            at += 1
    path = torch.stack([torch.randperm(t, generator=rng)[:n].sort().values for _ in range(s)])
    st = {"pages": pages, "k": _arena(case["cache"], pages, layers, elems, gen),
          "v": _arena(case["cache"], pages, layers, elems, gen), "tables": tables.int().to(DEV),
          "past": torch.tensor(past).int().to(DEV), "path": path.int().to(DEV),
          "n_path": torch.full((s,), n).int().to(DEV),
          "kc": torch.randn((layers, s * t, elems), generator=gen, device=DEV),
          "vc": torch.randn((layers, s * t, elems), generator=gen, device=DEV)}
    if own:
        st["cache_obj"] = _cache(case, pages, layers, st["k"], st["v"])
    return st


def _prepare_fork(case, seed, gen, rng):
    b, w, layers = case["batch"], case["beams"], case["layers"]
    elems, prefix = case["kv_heads"] * case["head_dim"], case["prefix"]
    # a request's beams share its prompt's pages, and have two pages of their own, the last one partial
    own_pages, free = 2, b * w + 2
    pages = b * (prefix + w * own_pages) + free
    order = torch.randperm(pages, generator=rng)
    tables, at = torch.empty((b * w, prefix + own_pages), dtype=torch.int64), 0
    lengths = torch.empty(b * w, dtype=torch.int64)
    refs = torch.zeros(pages, dtype=torch.int64)
    for i in range(b):
        shared = order[at:at + prefix]
        at += prefix
        refs[shared] += w
        fill = int(torch.randint(1, BLOCK, (1,), generator=rng))
        for j in range(w):
            tables[i * w + j, :prefix] = shared
            tables[i * w + j, prefix:] = order[at:at + own_pages]
            refs[order[at:at + own_pages]] += 1
            at += own_pages
            lengths[i * w + j] = (prefix + own_pages - 1) * BLOCK + fill
    parents = []
    for i in range(b):
        chosen = torch.randperm(w, generator=rng)[:case["survivors"]]
        extra = chosen[torch.randint(0, case["survivors"], (w - case["survivors"],), generator=rng)]
        mix = torch.cat([chosen, extra])[torch.randperm(w, generator=rng)]
        parents += (mix + i * w).tolist()
    st = {"pages": pages, "k": _arena(case["cache"], pages, layers, elems, gen),
          "v": _arena(case["cache"], pages, layers, elems, gen), "tables": tables.int().to(DEV),
          "lengths": lengths.int().to(DEV), "refs": refs.int().to(DEV), "parents": torch.tensor(parents).int().to(DEV)}
    if own:
        import densecore_amd as dc
        st["cache_obj"] = _cache(case, pages, layers, st["k"], st["v"])
        st["tables_out"], st["lengths_out"] = torch.empty_like(st["tables"]), torch.empty_like(st["lengths"])
        st["refs_out"], st["missing"] = torch.empty_like(st["refs"]), torch.empty(1, dtype=torch.int32, device=DEV)
        st["ws"] = torch.empty(max(dc.kv_fork_workspace_size(pages, b * w, b * w), 256), dtype=torch.uint8, device=DEV)
    return st


def _prepare_compact(case, seed, gen, rng):
    pages, live, moved, layers = case["pages"], case["live"], case["moved"], case["layers"]
    elems = case["kv_heads"] * case["head_dim"]
    held = torch.cat([torch.randperm(live, generator=rng)[:live - moved],
                      live + torch.randperm(pages - live, generator=rng)[:moved]])
    held = held[torch.randperm(live, generator=rng)]
    width = max(min(20, live), 1)
    seqs = (live + width - 1) // width
    tables, lengths = torch.full((seqs, width), -1), torch.empty(seqs, dtype=torch.int64)
    for i in range(seqs):
        mine = held[i * width:(i + 1) * width]
        tables[i, :len(mine)] = mine
        lengths[i] = len(mine) * BLOCK - int(torch.randint(0, BLOCK, (1,), generator=rng))
    refs = torch.zeros(pages, dtype=torch.int64)
    refs[held] = 1
    st = {"pages": pages, "k": _arena(case["cache"], pages, layers, elems, gen),
          "v": _arena(case["cache"], pages, layers, elems, gen), "tables": tables.int().to(DEV),
          "lengths": lengths.int().to(DEV), "refs": refs.int().to(DEV)}
    if own:
        import densecore_amd as dc
        st["cache_obj"] = _cache(case, pages, layers, st["k"], st["v"])
        st["tables_out"], st["refs_out"] = torch.empty_like(st["tables"]), torch.empty_like(st["refs"])
        st["n_live"] = torch.empty(1, dtype=torch.int32, device=DEV)
        st["ws"] = torch.empty(max(dc.kv_compact_workspace_size(pages), 256), dtype=torch.uint8, device=DEV)
    return st


def _prepare_beam(case, seed, gen, rng):
    rows, v = case["batch"] * case["beams"], case["vocab"]
    x = torch.randn((rows, v), generator=gen, device=DEV) * 3.0
    hot = torch.randint(0, v, (rows, 4), generator=gen, device=DEV)
    x.scatter_(1, hot, 9.0 + 2.0 * torch.randn((rows, 4), generator=gen, device=DEV))  # a model's few likely tokens
    x[:, :: 97] = -math.inf  # tokens that the program rules out
    st = {"x": x.half() if case["dtype"] == "F16" else x,
          "beam": -3.0 * torch.rand((case["batch"], case["beams"]), generator=gen, device=DEV)}
    if own:
        import densecore_amd as dc
        b, n = case["batch"], case["n_out"]
        st["scores"] = torch.empty((b, n), device=DEV)
        st["parents"], st["tokens"] = (torch.empty((b, n), dtype=torch.int32, device=DEV) for _ in range(2))
        need = dc.beam_select_workspace_size(b, case["beams"], v, n)
        st["ws"] = torch.empty(max(need, 256), dtype=torch.uint8, device=DEV)
    return st


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = torch.Generator()
    rng.manual_seed(seed + 1)
    make = {"tree": _prepare_tree, "path": _prepare_path, "fork": _prepare_fork, "compact": _prepare_compact,
            "beam": _prepare_beam}[case["op"]]
    return {"case": case, **make(case, seed, gen, rng)}


# ---------------------------------------------------------------- one pass
def _values(case, arena, pages, layers):
    """The arena's slots as values [pages, layers, 16, elems] (fp32, or the F16 / F32 storage itself)."""
    elems = case["kv_heads"] * case["head_dim"]
    if case["cache"] == "Q8_0":
        raw = arena.view(pages, layers, BLOCK, elems // 32, 34)
        d = raw[..., :2].contiguous().view(torch.float16).float()
        return (raw[..., 2:].view(torch.int8).float() * d).view(pages, layers, BLOCK, elems)
    dtype = torch.float16 if case["cache"] == "F16" else torch.float32
    return arena.view(dtype).view(pages, layers, BLOCK, elems)


def _slots(case, st, arena, ids):
    """fp32 rows [len(ids) * 16, kv_heads, head_dim] of the pages `ids` in the attended layer."""
    elems = case["kv_heads"] * case["head_dim"]
    raw = arena.view(st["pages"], st["layers"], BLOCK, -1)[ids, st["layer"]]
    one = {"cache": case["cache"], "kv_heads": case["kv_heads"], "head_dim": case["head_dim"]}
    return _values(one, raw.contiguous().view(-1), len(ids), 1).reshape(-1, case["kv_heads"], elems // case["kv_heads"]).float()


def _run_tree(st):
    case = st["case"]
    if own:
        return st["cache_obj"].tree_attention(st["layer"], st["tables"], st["past"], case["past_max"], st["q"], st["kc"],
                                              st["vc"], st["scale"], mask=st["mask"], n_draft=st["drafts"],
                                              out=st["out"], workspace=st["ws"])
    s, t, h, g, d = (case[x] for x in ("seqs", "tokens", "heads", "kv_heads", "head_dim"))
    rep = h // g
    out = torch.zeros((s, t, h * d), device=DEV)
    shift = torch.arange(t, device=DEV)
    for i, (past, n) in enumerate(zip(st["host_past"], st["host_drafts"])):
        ids = st["tables"][i, :(past + BLOCK - 1) // BLOCK].long()
        rows = slice(i * t, i * t + n)
        k = torch.cat([_slots(case, st, st["k"], ids)[:past], st["kc"][rows].view(n, g, d)]).permute(1, 0, 2)
        v = torch.cat([_slots(case, st, st["v"], ids)[:past], st["vc"][rows].view(n, g, d)]).permute(1, 0, 2)
        q = st["q"][rows].view(n, g, rep, d).permute(1, 0, 2, 3).reshape(g, n * rep, d)
        sc = torch.matmul(q, k.transpose(1, 2).contiguous()) * st["scale"]
        sees = (st["mask"][i, :n, shift[:n] // 64] >> (shift[:n] % 64)) & 1
        hidden = (sees == 0).repeat_interleave(rep, 0)
        sc[:, :, past:] = torch.where(hidden, torch.full((), -math.inf, device=DEV), sc[:, :, past:])
        p = torch.exp(sc - sc.amax(2, keepdim=True))
        o = torch.matmul(p, v.contiguous()) / p.sum(2, keepdim=True)
        out[i, :n] = o.view(g, n, rep, d).permute(1, 0, 2, 3).reshape(n, h * d)
    return out.view(s * t, h * d)


def _run_path(st):
    case = st["case"]
    if own:
        st["cache_obj"].write_path(st["tables"], st["past"], st["path"], st["n_path"], st["kc"], st["vc"])
    else:
        s, t, n = case["seqs"], case["tokens"], case["accepted"]
        pos = st["past"].long()[:, None] + torch.arange(n, device=DEV)
        page = torch.gather(st["tables"].long(), 1, pos // BLOCK).view(-1)
        src = (st["path"].long() + t * torch.arange(s, device=DEV)[:, None]).view(-1)
        for name, cur in (("k", st["kc"]), ("v", st["vc"])):
            a = _values(case, st[name], st["pages"], case["layers"])
            a[page, :, pos.view(-1) % BLOCK] = cur[:, src].transpose(0, 1).to(a.dtype)
    return [_values(case, st[x], st["pages"], case["layers"]) for x in ("k", "v")]


def _run_fork(st):
    case, n = st["case"], st["pages"]
    if own:
        out = st["cache_obj"].fork(st["tables"], st["lengths"], st["parents"], st["refs"], tables_out=st["tables_out"],
                                   lengths_out=st["lengths_out"], refs_out=st["refs_out"], missing=st["missing"],
                                   workspace=st["ws"])
        tables, lengths, refs, missing = out
    else:
        old, par = st["tables"].long(), st["parents"].long()
        at = torch.arange(old.shape[1], device=DEV)
        one = torch.ones((), dtype=torch.int64, device=DEV)
        holds = at < ((st["lengths"].long() + BLOCK - 1) // BLOCK)[:, None]
        lengths = st["lengths"].long()[par]
        tables, has = old[par], holds[par]
        refs = st["refs"].long().clone()
        refs.index_add_(0, old[holds], -one.expand(int(holds.sum())))
        refs.index_add_(0, tables[has], one.expand(int(has.sum())))
        child = torch.arange(len(par), device=DEV)
        partial = lengths % BLOCK != 0
        tail = torch.gather(tables, 1, (lengths // BLOCK).clamp(max=old.shape[1] - 1)[:, None])[:, 0]
        tail = torch.where(partial, tail, n)
        users = torch.zeros(n + 1, dtype=torch.int64, device=DEV).index_add_(0, tail, torch.ones_like(tail))
        first = torch.full((n + 1,), len(par), device=DEV).scatter_reduce_(0, tail, child, "amin")
        alone = torch.cat([refs, refs.new_zeros(1)])[tail] == users[tail]
        copies = partial & ~(alone & (first[tail] == child))
        free = torch.sort((refs > 0).long(), stable=True).indices
        rank = torch.cumsum(copies.long(), 0) - 1
        short = rank >= (refs == 0).sum()
        new = torch.where(short, -1, free[rank.clamp(0, n - 1)])
        who = copies.nonzero()[:, 0]
        refs.index_add_(0, tail[who], -torch.ones_like(who))
        got = who[new[who] >= 0]
        refs[new[got]] = 1
        tables = torch.where(has, tables, -1)
        tables[who, lengths[who] // BLOCK] = new[who]
        for name in ("k", "v"):
            a = st[name].view(n, -1)
            a[new[got]] = a[tail[got]]
        missing = (len(who) - len(got)) * one.view(1)
        tables, lengths, refs, missing = (x.int() for x in (tables, lengths, refs, missing))
    return [tables, lengths, refs, missing] + [_values(case, st[x], n, case["layers"]) for x in ("k", "v")]


def _run_compact(st):
    case, n = st["case"], st["pages"]
    if own:
        tables, refs, n_live = st["cache_obj"].compact(st["tables"], st["lengths"], st["refs"], tables_out=st["tables_out"],
                                                       refs_out=st["refs_out"], n_live=st["n_live"], workspace=st["ws"])
    else:
        refs, page = st["refs"].clone(), torch.arange(n, device=DEV)
        live = refs > 0
        n_live = live.sum().view(1).int()
        holes, movers = page[~live & (page < n_live)], page[live & (page >= n_live)]
        goes = page.clone()
        goes[movers] = holes
        for name in ("k", "v"):
            a = st[name].view(n, -1)
            a[holes] = a[movers]
        refs[holes] = st["refs"][movers]
        refs[movers] = 0
        holds = torch.arange(st["tables"].shape[1], device=DEV) < ((st["lengths"] + BLOCK - 1) // BLOCK)[:, None]
        tables = torch.where(holds, goes[st["tables"].long().clamp(min=0)].int(), st["tables"])
    return [tables, refs, n_live] + [_values(case, st[x], n, case["layers"]) for x in ("k", "v")]


def _run_beam(st):
    case = st["case"]
    if own:
        import densecore_amd as dc
        return list(dc.beam_select(st["x"], st["beam"], case["n_out"], scores=st["scores"], parents=st["parents"],
                                   tokens=st["tokens"], workspace=st["ws"]))
    b, w, v, n = case["batch"], case["beams"], case["vocab"], case["n_out"]
    x = st["x"].double()  # 64 bits: the order of candidates next to each other
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = (st["beam"].double().view(-1, 1) + (x - lse)).view(b, w * v)
    best = torch.sort(score, dim=1, descending=True, stable=True)
    val, idx = best.values[:, :n], best.indices[:, :n]
    if val.shape[1] < n:  # fewer candidates than asked for
        val = torch.cat([val, val.new_full((b, n - val.shape[1]), -math.inf)], 1)
        idx = torch.cat([idx, idx.new_zeros((b, n - idx.shape[1]))], 1)
    none = val == -math.inf
    row = idx // v + w * torch.arange(b, device=DEV)[:, None]
    return [val.float(), torch.where(none, -1, row).int(), torch.where(none, -1, idx % v).int()]


def run(state):
    return {"tree": _run_tree, "path": _run_path, "fork": _run_fork, "compact": _run_compact, "beam": _run_beam}[
        state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "beam":
        rows, v = case["batch"] * case["beams"], case["vocab"]
        size = 2 if case["dtype"] == "F16" else 4
        return {"bytes": rows * (v * size + 4) + case["batch"] * case["n_out"] * 12, "flops": 4 * rows * v}
    elems = case["kv_heads"] * case["head_dim"]
    slot = _row_bytes(case["cache"], elems)
    if op == "tree":
        t, hd = case["tokens"], case["heads"] * case["head_dim"]
        past, drafts = _pasts(case), _drafts(case)
        nbytes = sum(2 * p * slot + 4 * ((p + BLOCK - 1) // BLOCK) + 8 * n * (hd + elems) for p, n in zip(past, drafts))
        nbytes += case["seqs"] * t * 8 * ((t + 63) // 64) + 4 * hd * sum(t - n for n in drafts)
        return {"bytes": nbytes, "flops": sum(4 * n * hd * (p + n) for p, n in zip(past, drafts))}
    if op == "path":
        rows = case["seqs"] * case["accepted"] * case["layers"]
        return {"bytes": 2 * rows * (4 * elems + slot), "flops": 0}
    page = slot * case["layers"] * BLOCK
    if op == "fork":
        seqs, width = case["batch"] * case["beams"], case["prefix"] + 2
        copies = case["batch"] * (case["beams"] - case["survivors"])
        pages = case["batch"] * (case["prefix"] + 2 * case["beams"]) + seqs + 2
        return {"bytes": 4 * copies * page + 8 * (seqs * (width + 1) + pages) + 4 * seqs, "flops": 0}
    return {"bytes": 4 * case["moved"] * page + 8 * (case["pages"] + case["live"]), "flops": 0}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _decoded(case, raw):
    """Slot bytes [..., slot] -> float64 values [..., elems], each block by itself."""
    if case["cache"] == "Q8_0":
        blocks = raw.reshape(*raw.shape[:-1], -1, 34)
        scale = blocks[..., 0:2].clone(memory_format=torch.contiguous_format).view(torch.half).to(torch.float64)
        q = blocks[..., 2:].to(torch.float64)
        return (torch.where(q > 127, q - 256, q) * scale).flatten(-2)
    return raw.clone(memory_format=torch.contiguous_format).view(torch.half if case["cache"] == "F16" else torch.float32).to(
        torch.float64)


def _exact_tree(case, st):
    s, t, h, g, d = (case[x] for x in ("seqs", "tokens", "heads", "kv_heads", "head_dim"))
    out = torch.zeros((s, t, h, d), dtype=torch.float64, device=DEV)
    slot = _row_bytes(case["cache"], g * d)
    bits = st["mask"].cpu().tolist()
    for i in range(s):
        past, n = st["host_past"][i], st["host_drafts"][i]
        pos = torch.arange(past, device=DEV)
        line = (st["tables"][i].long()[pos // BLOCK] * st["layers"] + st["layer"]) * BLOCK + pos % BLOCK
        keys = [_decoded(case, st[x].view(-1, slot)[line]).view(past, g, d) for x in ("k", "v")]
        see = torch.ones((n, past + n), dtype=torch.bool)
        for a in range(n):
            for b in range(n):
                see[a, past + b] = (bits[i][a][b // 64] >> (b % 64)) & 1 == 1
        see = see.to(DEV)
        for head in range(h):
            kv = head // (h // g)
            k, v = (torch.cat([x[:, kv], c[i * t:i * t + n].view(n, g, d)[:, kv].double()])
                    for x, c in zip(keys, (st["kc"], st["vc"])))
            z = (st["q"][i * t:i * t + n].view(n, h, d)[:, head].double() @ k.T) * st["scale"]
            z = z.masked_fill(~see, -math.inf)
            out[i, :n, head] = torch.softmax(z, 1) @ v
    return out.view(s * t, h * d)


def _exact_path(case, st):
    res = []
    past, tables, path = (st[x].cpu().tolist() for x in ("past", "tables", "path"))
    for name, cur in (("k", st["kc"]), ("v", st["vc"])):
        slot = _row_bytes(case["cache"], cur.shape[2])
        a = _decoded(case, st[name].view(st["pages"], case["layers"], BLOCK, slot))
        for i in range(case["seqs"]):
            for j, tok in enumerate(path[i]):
                p = past[i] + j
                a[tables[i][p // BLOCK], :, p % BLOCK] = cur[:, i * case["tokens"] + tok].double()
        res.append(a)
    return res


def _exact_beam(case, st):
    b, w, v, n = case["batch"], case["beams"], case["vocab"], case["n_out"]
    scores = torch.full((b, n), -math.inf, dtype=torch.float64, device=DEV)
    for i in range(b):
        found = []
        for j in range(w):
            x = st["x"][i * w + j].to(torch.float64)
            lp = torch.log_softmax(x, 0) + float(st["beam"][i, j])
            found.append(torch.topk(lp, min(n, v)).values)
        best = torch.cat(found).sort(descending=True).values[:n]
        scores[i, :len(best)] = best
    return [scores, None, None]


def _moved(case, st, pairs):
    """The arenas' values after the copies of whole pages `pairs` = [(from, to)]."""
    slot = _row_bytes(case["cache"], case["kv_heads"] * case["head_dim"])
    res = []
    for name in ("k", "v"):
        a = _decoded(case, st[name].view(st["pages"], case["layers"], BLOCK, slot))
        for src, dst in pairs:
            a[dst] = a[src]
        res.append(a)
    return res


def _exact_fork(case, st):
    old, lens, refs, parents = (st[x].cpu().tolist() for x in ("tables", "lengths", "refs", "parents"))
    blocks = [-(-n // BLOCK) for n in lens]
    new = [old[p][:blocks[p]] for p in parents]
    for page in (e for t, n in zip(old, blocks) for e in t[:n]):
        refs[page] -= 1
    outside = list(refs)
    for page in (e for t in new for e in t):
        refs[page] += 1
    tails = [t[-1] if lens[p] % BLOCK else None for t, p in zip(new, parents)]
    full = {e for t, last in zip(new, tails) for e in (t if last is None else t[:-1])}
    free, pairs, kept = [p for p in range(len(refs)) if refs[p] == 0], [], set()
    for t, last in zip(new, tails):
        if last is None or (outside[last] == 0 and last not in full and last not in kept):
            kept.add(last)
            continue
        t[-1] = free.pop(0)
        refs[last] -= 1
        refs[t[-1]] += 1
        pairs.append((last, t[-1]))
    width = len(old[0])
    ints = [torch.tensor(x, device=DEV) for x in ([t + [-1] * (width - len(t)) for t in new], [lens[p] for p in parents],
                                                  refs, [0])]
    return ints + _moved(case, st, pairs)


def _exact_compact(case, st):
    tables, lens, refs = (st[x].cpu().tolist() for x in ("tables", "lengths", "refs"))
    live = sum(r > 0 for r in refs)
    pairs = list(zip((p for p in range(live, len(refs)) if refs[p] > 0), (p for p in range(live) if refs[p] == 0)))
    goes = dict(pairs)
    for src, dst in pairs:
        refs[dst], refs[src] = refs[src], 0
    for t, n in zip(tables, lens):
        for b in range(-(-n // BLOCK)):
            t[b] = goes.get(t[b], t[b])
    return [torch.tensor(x, device=DEV) for x in (tables, refs, [live])] + _moved(case, st, pairs)


def exact(case, seed):
    st = prepare(case, seed)
    return {"tree": _exact_tree, "path": _exact_path, "fork": _exact_fork, "compact": _exact_compact,
            "beam": _exact_beam}[case["op"]](case, st)
