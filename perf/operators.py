"""Operators for decoding several continuations of a prompt over an fp16 K/V cache.

Each case below is one operator of the framework at one size, in two forms: the
operator's formula in elementary torch operations (own = False) and the calls a
user makes of the framework (own = True).

  tree    q|k|v of drafted tokens rotated at their depth, k and v appended to the
          cache behind the committed positions, then attention of every node over
          the committed positions and its own ancestors among the nodes
  beam    the best continuations over beams x vocabulary
  fork    sequences continue their parents: page tables rewritten, partially
          filled pages copied, pages allocated for the positions to come
          (or, without a page table, rows copied between sequences)
  accept  the accepted nodes' K/V rows moved together behind the committed ones
"""
import math
import random

import torch

own = False

_DEVS = {}


def _dev(s):
    """The framework's device context on the stream of the state's first pass, torch's current one, which fills the inputs and
    reads the outputs; one a stream, kept for the process."""
    if "dev" not in s:
        at = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
        if at not in _DEVS:
            from prosperoai_b200.api import Device
            _DEVS[at] = Device(at[0], stream=at[1])
        s["dev"] = _DEVS[at]
    return s["dev"]


# ---- the cases --------------------------------------------------------------------------------------


def _tree(name, seqs, nodes, ragged, past, page, h, hk, hd):
    return {"name": name, "op": "tree", "seqs": seqs, "nodes": nodes, "ragged": ragged, "past": past, "page": page,
            "h": h, "hk": hk, "hd": hd}


def listed():
    return [
        # one token of one sequence over a prompt of 512: the smallest call of a decode loop, all latency
        _tree("one token at 512", 1, 1, False, 512, 0, 32, 8, 128),
        # a drafted tree of 16 over the 4096-position cache of one sequence
        _tree("tree of 16 at 4096", 1, 16, False, 4096, 0, 32, 8, 128),
        # one token each of 8 long sequences, in pages: the cache's bytes are all that counts
        _tree("8 x one token at 16384, paged", 8, 1, False, 16384, 128, 32, 8, 128),
        # a serving batch: sequences of 1 to 5001 positions with trees of 1 to 33 nodes
        _tree("8 ragged trees, paged", 8, 33, True, 5001, 128, 32, 8, 128),
        # large trees over long sequences: the tensor cores' work counts as much as the bytes
        _tree("8 x 64 nodes at 32768, paged", 8, 64, False, 32768, 128, 32, 8, 128),
        # the beams of one prompt over a small model's vocabulary
        {"name": "4 beams of 2048", "op": "beam", "prompts": 1, "beams": 4, "vocab": 2048, "pick": 4},
        # a batch of prompts over the 8B-shaped model's vocabulary, twice the beams kept as candidates
        {"name": "16 x 8 beams of 128256", "op": "beam", "prompts": 16, "beams": 8, "vocab": 128256, "pick": 16},
        # a beam step of a small model: a page or two to copy
        {"name": "fork 4 beams, 2 layers", "op": "fork", "groups": 1, "beams": 4, "len": 300, "page": 128, "layers": 2,
         "hk": 1, "hd": 128},
        # a beam step of the 8B-shaped model: the last, partly filled page of half the beams, in all layers
        {"name": "fork 8 beams, 32 layers", "op": "fork", "groups": 1, "beams": 8, "len": 700, "page": 128, "layers": 32,
         "hk": 8, "hd": 128},
        # the same where the cache is a session's, one run of positions for each sequence
        {"name": "fork 8 runs, 32 layers", "op": "fork", "groups": 1, "beams": 8, "len": 700, "page": 0, "layers": 32,
         "hk": 8, "hd": 128},
        # four accepted tokens of one sequence of a small model
        {"name": "accept 4, 2 layers", "op": "accept", "seqs": 1, "nodes": 16, "path": 4, "past": 300, "page": 128,
         "layers": 2, "hk": 1, "hd": 128},
        # six accepted tokens of each of 8 sequences, all layers of the 8B-shaped model
        {"name": "accept 8 x 6, 32 layers", "op": "accept", "seqs": 8, "nodes": 33, "path": 6, "past": 700, "page": 128,
         "layers": 32, "hk": 8, "hd": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "beam", "fork", "accept"])
    if op == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 13])
        prompts = _log(rng, 1, max(1, 128 // beams))
        return {"op": op, "prompts": prompts, "beams": beams, "vocab": _log(rng, 300, 128256),
                "pick": rng.choice([beams, 2 * beams])}
    h, hk, hd = rng.choice([(32, 8, 128), (16, 2, 128), (8, 8, 128), (2, 1, 128), (32, 8, 64), (14, 2, 64)])
    if op == "tree":
        seqs = _log(rng, 1, 16)
        past = _log(rng, 1, 262144 // seqs)
        nodes = _log(rng, 1, 64)
        return {"op": op, "seqs": seqs, "nodes": nodes, "ragged": rng.random() < 0.5, "past": past,
                "page": rng.choice([0, 16, 64, 128, 128]), "h": h, "hk": hk, "hd": hd}
    layers = rng.choice([1, 2, 5, 32])
    if op == "fork":
        groups, beams, page = rng.choice([1, 2, 3]), rng.choice([2, 3, 4, 5, 8]), rng.choice([0, 16, 64, 128, 128])
        return {"op": op, "groups": groups, "beams": beams, "len": _log(rng, 1, 700 // groups), "page": page,
                "layers": layers, "hk": hk, "hd": hd}
    nodes = rng.randint(1, 64)
    return {"op": op, "seqs": rng.randint(1, 8), "nodes": nodes, "path": rng.randint(1, 1 + nodes // 3),
            "past": _log(rng, 1, 700), "page": rng.choice([0, 16, 64, 128, 128]), "layers": layers, "hk": hk, "hd": hd}


# ---- inputs -----------------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62) + 1)
    return g


def _dims(case):
    """(lengths, node counts) of a tree case's sequences; the same for every seed."""
    r = random.Random(case["seqs"] * 1000003 + case["past"] * 101 + case["nodes"])
    if not case["ragged"]:
        return [case["past"]] * case["seqs"], [case["nodes"]] * case["seqs"]
    lens = [max(1, int(case["past"] * r.random() ** 2)) for _ in range(case["seqs"])]
    nodes = [r.randint(1, case["nodes"]) for _ in range(case["seqs"])]
    lens[-1], nodes[0] = case["past"], case["nodes"]
    return lens, nodes


def _tree_of(r, n):
    """A drafted tree's (depth, mask words) of n nodes in breadth-first order: parents come from the last 8 nodes."""
    depth, bits = [0], [1]
    for i in range(1, n):
        p = r.randint(max(0, i - 8), i - 1)
        depth.append(depth[p] + 1)
        bits.append(bits[p] | 1 << i)
    return depth, bits


def _cache(g, layers, pages, hk, tokens, hd):
    return [torch.randn(layers, pages, hk, tokens, hd, generator=g, device="cuda", dtype=torch.float16) for _ in range(2)]


def _pages(g, rows, page, spare=0):
    """Page tables of sequences that need `rows` positions: shuffled pages, -1 behind them, `spare` pages in no table."""
    need = [-(-n // page) for n in rows]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(rows), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    return table, total


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return {"tree": _prepare_tree, "beam": _prepare_beam, "fork": _prepare_fork, "accept": _prepare_accept}[case["op"]](case, seed)


def _prepare_tree(c, seed):
    g, r = _gen(seed), random.Random(seed)
    lens, nodes = _dims(c)
    h, hk, hd, n_seq, rows = c["h"], c["hk"], c["hd"], c["seqs"], sum(nodes)
    most, words = max(nodes), -(-max(nodes) // 64)
    depth, mask = [], []
    for n in nodes:
        d, bits = _tree_of(r, n)
        depth += d
        mask += [[(b >> 64 * w & (1 << 64) - 1) for w in range(words)] for b in bits]
    mask = [[w - (1 << 64) if w >> 63 else w for w in m] for m in mask]
    if c["page"]:
        table, n_pages = _pages(g, [a + b for a, b in zip(lens, nodes)], c["page"])
        page = c["page"]
    else:
        page = -(-(max(lens) + most) // 128) * 128
        table, n_pages = None, n_seq
    k, v = _cache(g, 1, n_pages, hk, page, hd)
    top = max(lens) + most
    inv = 500000.0 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))
    ang = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * inv
    off = [0]
    for n in nodes:
        off.append(off[-1] + n)
    return {"case": c, "k": k, "v": v, "table": table, "page": page, "n_pages": n_pages, "rows": rows, "most": most,
            "lens": _i32(lens), "off": _i32(off), "depth": _i32(depth),
            "mask": torch.tensor(mask, dtype=torch.int64, device="cuda"),
            "seq": torch.tensor([s for s, n in enumerate(nodes) for _ in range(n)], device="cuda"),
            "node": torch.tensor([i for n in nodes for i in range(n)], device="cuda"),
            "cos": ang.cos().float(), "sin": ang.sin().float(),
            "qkv": torch.randn(rows, h + 2 * hk, hd, generator=g, device="cuda"),
            "q": torch.empty(rows, h, hd, device="cuda"), "out": torch.empty(rows, h, hd, device="cuda")}


def _prepare_beam(c, seed):
    g, r = _gen(seed), random.Random(seed)
    n, b, vocab = c["prompts"], c["beams"], c["vocab"]
    # a language model's logits: a few tokens of a row stand out
    logits = torch.randn(n, b, vocab, generator=g, device="cuda") * 3
    done = [[int(b > 1 and r.random() < 0.1) for _ in range(b)] for _ in range(n)]
    return {"case": c, "logits": logits, "scores": -6 * torch.rand(n, b, generator=g, device="cuda"), "done": _i32(done),
            "pad": 2 % vocab, "out_scores": torch.empty(n, c["pick"], device="cuda"),
            "out_parents": torch.empty(n, c["pick"], dtype=torch.int32, device="cuda"),
            "out_tokens": torch.empty(n, c["pick"], dtype=torch.int32, device="cuda")}


def _fork_plan(c):
    """(parents, copied sequences) of a fork case: every other beam ends, its neighbour's continuation takes its place."""
    par = [i - (i % c["beams"]) % 2 for i in range(c["groups"] * c["beams"])]
    return par, sum(p != i for i, p in enumerate(par))


def _prepare_fork(c, seed):
    g = _gen(seed)
    n_seq, ln, page = c["groups"] * c["beams"], c["len"], c["page"]
    parents, _ = _fork_plan(c)
    if page:
        # the beams of a prompt share its full pages and own their last one
        full, rest = ln // page, int(ln % page > 0)
        width = full + 2
        total = c["groups"] * full + n_seq * (rest + 1)
        perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        table = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
        for s in range(n_seq):
            q = s // c["beams"]
            table[s, :full] = perm[q * full:(q + 1) * full]
            if rest:
                table[s, full] = perm[c["groups"] * full + s]
        tokens, pages = page, total
    else:
        tokens, pages, table, width = -(-(ln + 1) // 128) * 128, n_seq, None, 1
    k, v = _cache(g, c["layers"], pages, c["hk"], tokens, c["hd"])
    return {"case": c, "k": k, "v": v, "table": table, "page": tokens, "n_pages": pages, "lens": _i32([ln] * n_seq),
            "parents": _i32(parents), "grow": _i32([1] * n_seq),
            "table_out": torch.empty(n_seq, width, dtype=torch.int32, device="cuda"),
            "lens_out": torch.empty(n_seq, dtype=torch.int32, device="cuda"),
            "granted": torch.empty(n_seq, dtype=torch.int32, device="cuda")}


def _prepare_accept(c, seed):
    g, r = _gen(seed), random.Random(seed)
    n_seq, page, most = c["seqs"], c["page"], c["path"]
    # a path's nodes behind its first: none of them lies where an accepted row goes
    paths = [[0] + sorted(r.sample(range(most, c["nodes"]), most - 1)) for _ in range(n_seq)]
    if page:
        table, pages = _pages(g, [c["past"] + c["nodes"]] * n_seq, page)
    else:
        page, table, pages = -(-(c["past"] + c["nodes"]) // 128) * 128, None, n_seq
    k, v = _cache(g, c["layers"], pages, c["hk"], page, c["hd"])
    return {"case": c, "k": k, "v": v, "table": table, "page": page, "n_pages": pages, "lens": _i32([c["past"]] * n_seq),
            "path": _i32(paths), "n_path": _i32([most] * n_seq),
            "lens_out": torch.empty(n_seq, dtype=torch.int32, device="cuda")}


# ---- one pass ---------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tree": _own_tree, "beam": _own_beam, "fork": _own_fork, "accept": _own_accept}[op](state)
    return {"tree": _plain_tree, "beam": _plain_beam, "fork": _plain_fork, "accept": _plain_accept}[op](state)


def _view(s):
    """The framework's description of the state's cache, made once and kept beside it."""
    if "view" not in s:
        from prosperoai_b200.api import KvView
        k = s["k"]
        s["view"] = KvView.of(k.data_ptr(), s["v"].data_ptr(), n_layer=k.shape[0], n_seq=s["lens"].numel(),
                              kv_heads=k.shape[2], head_dim=k.shape[4], page_tokens=s["page"], n_pages=s["n_pages"],
                              table=None if s["table"] is None else s["table"].data_ptr(),
                              max_pages=1 if s["table"] is None else s["table"].shape[1])
    return s["view"]


def _own_tree(s):
    dev, kv, h = _dev(s), _view(s), s["case"]["h"]
    lens, off, q = s["lens"].data_ptr(), s["off"].data_ptr(), s["q"].data_ptr()
    dev.rope_append(kv, 0, h, s["rows"], s["most"], lens, off, s["depth"].data_ptr(), s["qkv"].data_ptr(),
                    s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], q)
    dev.attn_tree(kv, 0, h, s["rows"], s["most"], lens, off, s["mask"].data_ptr(), q, s["out"].data_ptr())
    return {"out": s["out"], "k": s["k"], "v": s["v"]}


def _own_beam(s):
    c = s["case"]
    _dev(s).beam_select(c["prompts"], c["beams"], c["vocab"], s["logits"].data_ptr(), c["vocab"], s["scores"].data_ptr(),
                        s["done"].data_ptr(), s["pad"], c["pick"], s["out_scores"].data_ptr(),
                        s["out_parents"].data_ptr(), s["out_tokens"].data_ptr())
    return {"scores": s["out_scores"], "parents": s["out_parents"], "tokens": s["out_tokens"]}


def _own_fork(s):
    paged = s["table"] is not None
    _dev(s).kv_fork(_view(s), 0, s["lens"].data_ptr(), s["parents"].data_ptr(), s["grow"].data_ptr(),
                    s["table_out"].data_ptr() if paged else None, s["lens_out"].data_ptr(), s["granted"].data_ptr())
    return _forked(s)


def _forked(s):
    out = {"k": s["k"], "v": s["v"], "lens": s["lens_out"], "granted": s["granted"]}
    return out if s["table"] is None else {**out, "table": s["table_out"]}


def _own_accept(s):
    _dev(s).kv_accept(_view(s), s["path"].shape[1], s["lens"].data_ptr(), s["path"].data_ptr(), s["n_path"].data_ptr(),
                      s["lens_out"].data_ptr())
    return {"k": s["k"], "v": s["v"], "lens": s["lens_out"]}


def _slot(s, seq, pos):
    """(page, row of the page) of positions of sequences."""
    page = seq if s["table"] is None else s["table"][seq, pos // s["page"]].long()
    return page, pos % s["page"]


def _plain_tree(s):
    c = s["case"]
    h, hk, hd, n_seq, most = c["h"], c["hk"], c["hd"], c["seqs"], s["most"]
    seq, node, lens = s["seq"], s["node"], s["lens"].long()
    # rotate q and k at the node's position, append k and v
    at = lens[seq] + s["depth"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    x0, x1 = s["qkv"][:, :h + hk, :hd // 2], s["qkv"][:, :h + hk, hd // 2:]
    rot = torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1)
    page, row = _slot(s, seq, lens[seq] + node)
    s["k"][0, page, :, row] = rot[:, h:].half()
    s["v"][0, page, :, row] = s["qkv"][:, h + hk:].half()
    # attention: [sequence][kv head][node x query head of the group] against every position of the table
    if s["table"] is None:
        k, v = s["k"][0], s["v"][0]
    else:
        at = s["table"].clamp(min=0).long()
        k, v = (x[0][at].transpose(1, 2).reshape(n_seq, hk, -1, hd) for x in (s["k"], s["v"]))
    npos = k.shape[2]
    q = torch.zeros(n_seq, most, hk, h // hk, hd, device=rot.device)
    q[seq, node] = rot[:, :h].reshape(-1, hk, h // hk, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(n_seq, hk, -1, hd)
    score = (q @ k.float().transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).view(n_seq, hk, most, h // hk, npos)
    pos = torch.arange(npos, device=rot.device)
    behind = pos - lens[:, None]  # [sequence][position]: the node at this position, below 0 for a committed one
    bits = torch.zeros(n_seq, most, s["mask"].shape[1], dtype=torch.int64, device=rot.device)
    bits[seq, node] = s["mask"]
    inside = (behind >= 0) & (behind < most)
    j = behind.clamp(0, most - 1)
    word = torch.gather(bits, 2, (j // 64)[:, None].expand(-1, most, -1))
    seen = (behind < 0)[:, None] | inside[:, None] & ((word >> (j % 64)[:, None]) & 1).bool()
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(n_seq, hk, -1, npos) @ v.float()
    o = o.view(n_seq, hk, most, h // hk, hd) / torch.where(total == 0, 1.0, total)
    out = o.permute(0, 2, 1, 3, 4).reshape(n_seq, most, h, hd)[seq, node]
    return {"out": out, "k": s["k"], "v": s["v"]}


def _plain_beam(s):
    c = s["case"]
    n, b, vocab, pick = c["prompts"], c["beams"], c["vocab"], c["pick"]
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    z = torch.where(x == top, 0.0, x - top)
    logp = z - z.exp().sum(-1, keepdim=True).log()
    logp = torch.where(top == -math.inf, -math.inf, logp)
    start = s["scores"].double()[..., None]
    stay = torch.where(torch.arange(vocab, device=x.device) == s["pad"], start, -math.inf)
    cand = torch.where(s["done"][..., None] != 0, stay, start + logp).view(n, b * vocab)
    cand = torch.where(cand.isnan(), -math.inf, cand)
    # equal scores: the lowest flat index first
    best, at = cand.sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :pick], at[:, :pick]
    none = best == -math.inf
    first = torch.arange(n, device=x.device)[:, None] * b
    return {"scores": best.float(), "parents": torch.where(none, -1, first + at // vocab).int(),
            "tokens": torch.where(none, s["pad"], at % vocab).int()}


def _plain_fork(s):
    lens, parents, grow, page = s["lens"].long(), s["parents"].long(), s["grow"].long(), s["page"]
    n_seq, dev = lens.numel(), lens.device
    live = (parents >= 0) & (parents < n_seq)
    p = parents.clamp(0, n_seq - 1)
    ln = torch.where(live, lens[p], 0)
    grow = torch.where(live, grow, 0)
    if s["table"] is None:
        rows = int(s["case"]["len"])
        for x in (s["k"], s["v"]):
            x[:, :, :, :rows] = x[:, p, :, :rows]
        granted = torch.where(ln + grow <= page, grow, 0)
        s["lens_out"].copy_(ln)
        s["granted"].copy_(granted)
        return _forked(s)
    width, n_pages = s["table"].shape[1], s["n_pages"]
    col = torch.arange(width, device=dev)
    used = (ln + page - 1) // page
    held = col < used[:, None]
    new = torch.where(held, s["table"][p].long(), -1)
    # a page's rows in use, by the sequence that uses most of it
    ext = torch.where(held, (ln[:, None] - col * page).clamp(max=page), 0)
    most = torch.zeros(n_pages + 1, dtype=torch.int64, device=dev)
    most.scatter_reduce_(0, new.reshape(-1) % (n_pages + 1), ext.reshape(-1), "amax")
    last = new.gather(1, (used - 1).clamp(min=0)[:, None])[:, 0]
    mine = ln % page
    writes = (grow > 0) & (mine > 0) & (last >= 0)
    at = torch.arange(n_seq, device=dev)
    most_of = most[last.clamp(min=0)]
    keeper = torch.full((n_pages + 1,), n_seq, dtype=torch.int64, device=dev)
    keeper.scatter_reduce_(0, torch.where(writes & (mine == most_of), last, n_pages), at, "amin")
    fits = ln + grow <= width * page
    copy = writes & fits & (keeper[last.clamp(min=0)] != at)
    want = torch.where(fits & (grow > 0), (ln + grow + page - 1) // page - used, 0) + copy
    free = most[:n_pages] == 0
    order = free.sort(descending=True, stable=True)[1]  # the free pages, lowest first
    end = want.cumsum(0)
    ok = fits & ((want == 0) | (end <= free.sum()))
    copy, got = copy & ok, torch.where(ok, want, 0)
    begin = end - want
    fresh = torch.where(ok & (grow > 0), (ln + grow + page - 1) // page, used)
    nth = begin[:, None] + copy[:, None] + col - used[:, None]
    take = (col >= used[:, None]) & (col < fresh[:, None])
    new = torch.where(take, order[nth.clamp(0, n_pages - 1)], new)
    dst = order[begin.clamp(0, n_pages - 1)]
    new = torch.where(copy[:, None] & (col == used[:, None] - 1), dst[:, None], new)
    # the copies: rows of the partly filled page that are in use
    src, dst = torch.where(copy, last, 0), torch.where(copy, dst, 0)
    move = (torch.arange(page, device=dev) < mine[:, None]) & copy[:, None]
    seq, row = move.nonzero(as_tuple=True)
    for x in (s["k"], s["v"]):
        x[:, dst[seq], :, row] = x[:, src[seq], :, row]
    s["table_out"].copy_(new)
    s["lens_out"].copy_(ln)
    s["granted"].copy_(torch.where(ok, grow, 0))
    return _forked(s)


def _plain_accept(s):
    lens, path, n_path = s["lens"].long(), s["path"].long(), s["n_path"].long()
    n_seq, most = path.shape
    i = torch.arange(most, device=path.device)
    seq = torch.arange(n_seq, device=path.device)[:, None].expand(-1, most)
    src, dst = _slot(s, seq, lens[:, None] + path), _slot(s, seq, lens[:, None] + i)
    move = i < n_path[:, None]
    for x in (s["k"], s["v"]):
        old = x[:, dst[0], :, dst[1]]
        x[:, dst[0], :, dst[1]] = torch.where(move[..., None, None, None], x[:, src[0], :, src[1]], old)
    s["lens_out"].copy_(lens + n_path)
    return {"k": s["k"], "v": s["v"], "lens": s["lens_out"]}


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "tree":
        lens, nodes = _dims(c)
        rows = sum(nodes)
        cached = sum(lens) * c["hk"] * c["hd"] * 2 * 2
        new = rows * c["hk"] * c["hd"] * 2 * 2
        return {"bytes": cached + new + rows * (2 * c["h"] + 2 * c["hk"]) * c["hd"] * 4 + rows * c["hd"] * 4,
                "flops": sum(4 * n * c["h"] * c["hd"] * (m + (n + 1) / 2) for m, n in zip(lens, nodes))}
    if c["op"] == "beam":
        n = c["prompts"] * c["beams"] * c["vocab"]
        return {"bytes": n * 4 + c["prompts"] * (c["beams"] * 8 + c["pick"] * 12), "flops": 3 * n}
    row = c["layers"] * c["hk"] * c["hd"] * 2 * 2
    if c["op"] == "fork":
        copied = _fork_plan(c)[1]
        n_seq = c["groups"] * c["beams"]
        if c["page"]:
            return {"bytes": copied * (c["len"] % c["page"]) * row * 2 + n_seq * (c["len"] // c["page"] + 2) * 8 + n_seq * 20,
                    "flops": 0}
        return {"bytes": copied * c["len"] * row * 2 + n_seq * 20, "flops": 0}
    return {"bytes": c["seqs"] * (c["path"] - 1) * row * 2 + c["seqs"] * (c["path"] + 3) * 4, "flops": 0}


# ---- the definitions in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "beam": _exact_beam, "fork": _exact_fork, "accept": _exact_accept}[case["op"]](s)


def _where(s, seq, pos):
    return (seq, pos) if s["table"] is None else (int(s["table"][seq, pos // s["page"]]), pos % s["page"])


def _exact_tree(s):
    c = s["case"]
    h, hk, hd, g = c["h"], c["hk"], c["hd"], c["h"] // c["hk"]
    kc, vc, x = s["k"][0], s["v"][0], s["qkv"].double()
    outs, off, lens, depth = [], s["off"].tolist(), s["lens"].tolist(), s["depth"].tolist()
    r2 = hd // 2
    for q in range(c["seqs"]):
        lo, hi, past = off[q], off[q + 1], lens[q]
        at = torch.tensor([past + depth[r] for r in range(lo, hi)], device=x.device)
        cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
        a, b = x[lo:hi, :, :r2], x[lo:hi, :, r2:]
        rot = torch.empty_like(x[lo:hi])
        rot[..., :r2] = a * cos - b * sin
        rot[..., r2:] = a * sin + b * cos
        for i in range(hi - lo):
            page, row = _where(s, q, past + i)
            kc[page, :, row] = rot[i, h:h + hk].half()
            vc[page, :, row] = x[lo + i, h + hk:].half()
        n = past + hi - lo
        if s["table"] is None:
            key, val = kc[q, :, :n].double(), vc[q, :, :n].double()
        else:
            need = s["table"][q, :-(-n // s["page"])].long()
            key, val = (t[need].double().permute(1, 0, 2, 3).reshape(hk, -1, hd)[:, :n] for t in (kc, vc))
        sees = torch.ones(hi - lo, n, dtype=torch.bool, device=x.device)
        for j in range(hi - lo):
            sees[:, past + j] = (s["mask"][lo:hi, j // 64] >> (j % 64)) & 1 == 1
        qh = rot[:, :h].reshape(-1, hk, g, hd)
        sc = torch.einsum("nkgd,kpd->kngp", qh, key) * hd ** -0.5
        sc = torch.where(sees[None, :, None], sc, torch.tensor(-math.inf, dtype=sc.dtype, device=sc.device))
        outs.append(torch.einsum("kngp,kpd->nkgd", torch.softmax(sc, -1), val).reshape(-1, h, hd))
    return {"out": torch.cat(outs), "k": s["k"].double(), "v": s["v"].double()}


def _exact_beam(s):
    x = s["logits"].double()
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    pad, n, b = s["pad"], x.shape[0], x.shape[1]
    best = []
    for i in range(n):
        cand = []
        for j in range(b):
            start = float(s["scores"][i, j])
            if int(s["done"][i, j]):
                cand.append(torch.tensor([start], dtype=torch.float64, device=x.device))
            else:
                cand.append(start + torch.topk(logp[i, j], min(s["case"]["pick"], x.shape[2])).values)
        cand.append(torch.full((s["case"]["pick"],), -math.inf, dtype=torch.float64, device=x.device))
        best.append(torch.topk(torch.cat(cand), s["case"]["pick"]).values)
    return {"scores": torch.stack(best), "parents": None, "tokens": None}


def _exact_fork(s):
    c = s["case"]
    parents, page, ln = s["parents"].tolist(), s["page"], c["len"]
    k, v = s["k"].clone(), s["v"].clone()
    if s["table"] is None:
        for i, p in enumerate(parents):
            for new, old in ((k, s["k"]), (v, s["v"])):
                new[:, i, :, :ln] = old[:, p, :, :ln]
        return {"k": k.double(), "v": v.double(), "lens": None, "granted": None}
    rows = ln % page
    table, used = s["table"].tolist(), -(-ln // page)
    held = {table[p][j] for p in parents for j in range(used)}
    free = [i for i in range(s["n_pages"]) if i not in held]
    kept = set()
    for p in parents:
        last = table[p][used - 1]
        if rows and last in kept:
            to = free.pop(0)
            for new, old in ((k, s["k"]), (v, s["v"])):
                new[:, to, :, :rows] = old[:, last, :, :rows]
        elif not rows:
            free.pop(0)
        kept.add(last)
    return {"k": k.double(), "v": v.double(), "table": None, "lens": None, "granted": None}


def _exact_accept(s):
    k, v = s["k"].clone(), s["v"].clone()
    for q, (past, path, n) in enumerate(zip(s["lens"].tolist(), s["path"].tolist(), s["n_path"].tolist())):
        for i in range(n):
            (p0, r0), (p1, r1) = _where(s, q, past + path[i]), _where(s, q, past + i)
            k[:, p1, :, r1] = s["k"][:, p0, :, r0]
            v[:, p1, :, r1] = s["v"][:, p0, :, r0]
    return {"k": k.double(), "v": v.double(), "lens": None}
