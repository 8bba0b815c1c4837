"""The operators of several continuations of one request, as cases to time: drafted trees and beams over the paged cache.

Kinds of case (`"kind"`):
  tree    attention of a batch of drafted token trees over a paged cache (`ops.tree_attention`): the drafted tokens' keys and values
          stand in the cache behind the request's own, and a token sees all of those and its ancestors in the tree
  keep    after a tree is verified: the accepted path's rows move up, side by side, in every layer's cache (`ops.compact_rows`)
  copy    blocks of a cache copied in all layers at once (`ops.copy_blocks`): the last, partly filled pages of forked requests, or
          the fixed-size states of the requests that surviving beams pass on
  beam    a step's choice over beams and vocabulary (`ops.beam_select`): scores, origins and tokens of the best continuations

Layer, head and vocabulary sizes are those of the models that `bench.py` measures.
"""
import math
import random

import numpy as np
import torch

own = False

VOCAB = 151936
LAYERS = 36


def listed():
    return [
        # one user's chat: sixteen drafted tokens behind two thousand, where launches and the start of the kernel count
        {"name": "tree_1x16", "kind": "tree", "requests": 1, "tokens": 16, "context": 2000, "heads": 32, "groups": 8, "dim": 128,
         "page": 64, "window": 0, "cap": 0.0, "sink": False, "dtype": "bfloat16"},
        # a few users with contexts and trees of all lengths, on the engine's small pages
        {"name": "tree_8x32_ragged", "kind": "tree", "requests": 8, "tokens": 32, "context": 8000, "heads": 32, "groups": 8, "dim": 128,
         "page": 16, "window": 0, "cap": 0.0, "sink": False, "dtype": "bfloat16"},
        # a loaded server with large trees: every head group's rows fill two tiles of the tensor cores
        {"name": "tree_32x64", "kind": "tree", "requests": 32, "tokens": 64, "context": 8192, "heads": 32, "groups": 8, "dim": 128,
         "page": 64, "window": 0, "cap": 0.0, "sink": False, "dtype": "bfloat16"},
        # one very long document
        {"name": "tree_1x64_long", "kind": "tree", "requests": 1, "tokens": 64, "context": 131001, "heads": 32, "groups": 8, "dim": 128,
         "page": 64, "window": 0, "cap": 0.0, "sink": False, "dtype": "bfloat16"},
        # small heads with a window, capped scores and a sink
        {"name": "tree_6x21_window", "kind": "tree", "requests": 6, "tokens": 21, "context": 5000, "heads": 16, "groups": 4, "dim": 64,
         "page": 16, "window": 1024, "cap": 30.0, "sink": True, "dtype": "bfloat16"},
        # the 32-bit path
        {"name": "tree_2x15_float32", "kind": "tree", "requests": 2, "tokens": 15, "context": 1500, "heads": 16, "groups": 8, "dim": 128,
         "page": 16, "window": 0, "cap": 0.0, "sink": False, "dtype": "float32"},
        # the accepted path of one user's tree, and of a full batch of large trees
        {"name": "keep_1", "kind": "keep", "requests": 1, "tokens": 16, "most": 5, "groups": 8, "dim": 128, "page": 64, "dtype": "bfloat16"},
        {"name": "keep_64", "kind": "keep", "requests": 64, "tokens": 64, "most": 9, "groups": 8, "dim": 128, "page": 64,
         "dtype": "bfloat16"},
        # one prompt goes on in eight beams: its last page, partly filled, is copied seven times
        {"name": "copy_pages_7", "kind": "copy", "moves": 7, "pieces": 8, "rows": 64, "row_bytes": 256, "arrays": 72, "blocks": 160,
         "whole": False},
        # the states of a recurrent decoder's layers, 32 running beams of which 19 are replaced
        {"name": "copy_states_19", "kind": "copy", "moves": 19, "pieces": 1, "rows": 1, "row_bytes": 1048576, "arrays": 36, "blocks": 32,
         "whole": True},
        # one prompt with four beams, and sixteen with eight
        {"name": "beam_1x4", "kind": "beam", "prompts": 1, "beams": 4, "choices": 8, "vocab": VOCAB, "first": False},
        {"name": "beam_16x8", "kind": "beam", "prompts": 16, "beams": 8, "choices": 16, "vocab": VOCAB, "first": False},
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(["tree", "tree", "tree", "keep", "copy", "beam"])
    if kind == "tree":
        dtype = rng.choice(["bfloat16"] * 4 + ["float32"])
        dim = rng.choice([64, 128, 128])
        groups = rng.choice([2, 4, 8])
        case = {"kind": kind, "requests": spread(1, 32), "tokens": spread(1, 128), "context": spread(1, 32000),
                "heads": groups * rng.choice([1, 2, 4, 5, 8]), "groups": groups, "dim": dim, "page": rng.choice([16, 64]),
                "window": rng.choice([0, 0, 0, spread(64, 4096)]), "cap": rng.choice([0.0, 0.0, 0.0, 30.0]),
                "sink": rng.random() < 0.25, "dtype": dtype}
        # no more than the largest listed case: keys and values read, and products of rows and keys
        while case["requests"] > 1 and case["requests"] * case["context"] * groups * dim > 32 * 8192 * 8 * 128 // (2 if dtype == "float32" else 1):
            case["requests"] //= 2
        most = 32 * 64 * 32 * 8192 * 128 // (24 if dtype == "float32" else 1)
        while case["requests"] > 1 and case["requests"] * case["tokens"] * case["heads"] * case["context"] * dim > most:
            case["requests"] //= 2
        while case["tokens"] * case["heads"] * case["context"] * dim > most:
            case["context"] //= 2
        return case
    if kind == "keep":
        return {"kind": kind, "requests": spread(1, 64), "tokens": rng.randint(18, 64), "most": rng.randint(1, 9), "groups": rng.choice([2, 4, 8]),
                "dim": rng.choice([64, 128]), "page": rng.choice([16, 64]), "dtype": rng.choice(["bfloat16", "float32"])}
    if kind == "copy":
        if rng.random() < 0.5:
            return {"kind": kind, "moves": spread(1, 60), "pieces": rng.choice([2, 4, 8]), "rows": rng.choice([16, 64]),
                    "row_bytes": rng.choice([128, 256, 512]), "arrays": 2 * rng.randint(4, 36), "blocks": 160, "whole": False}
        return {"kind": kind, "moves": spread(1, 31), "pieces": 1, "rows": 1, "row_bytes": rng.choice([9216, 65536, 262148, 1048576]),
                "arrays": rng.randint(4, 36), "blocks": 64, "whole": True}
    beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
    return {"kind": kind, "prompts": spread(1, 128 // beams), "beams": beams, "choices": 2 * beams, "vocab": spread(500, VOCAB),
            "first": rng.random() < 0.2}


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Cached tokens and drafted tokens of every request: the first has the most of both, the others anything down to a few."""
    r = random.Random(repr(sorted(case.items(), key=lambda kv: kv[0])))
    contexts, tokens = [case["context"]], [case["tokens"]]
    for _ in range(case["requests"] - 1):
        contexts.append(max(1, int(case["context"] * r.uniform(0.1, 1.0))))
        tokens.append(max(1, int(case["tokens"] * r.uniform(0.3, 1.0))))
    return contexts, tokens


def _tree_parents(n, r):
    """The parents of a drafted tree in the order of its rows: the best continuations go deep, the others branch off."""
    return [-1] + [i - 1 if r.random() < 0.4 else r.randrange(max(0, i - 12), i) for i in range(1, n)]


def _prepare_tree(case, seed):
    dev, dt = "cuda", getattr(torch, case["dtype"])
    r = random.Random(seed)
    contexts, tokens = _lengths(case)
    R, H, G, hd, pt = case["requests"], case["heads"], case["groups"], case["dim"], case["page"]
    n, most_tokens = sum(tokens), max(tokens)
    most_keys = max(c + t for c, t in zip(contexts, tokens))
    words = -(-most_tokens // 32)
    need = [-(-(c + t) // pt) for c, t in zip(contexts, tokens)]
    num_pages = sum(need) + 3
    order = np.random.RandomState(seed % (1 << 32)).permutation(num_pages)
    table = np.full((R, max(need)), -1, dtype=np.int32)
    requests = np.zeros((R, 4), dtype=np.int32)
    ancestors = np.zeros((n, words), dtype=np.uint32)
    positions = np.zeros(n, dtype=np.int32)
    at = row = 0
    for i in range(R):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        requests[i] = (i, row, tokens[i], contexts[i])
        for j, p in enumerate(_tree_parents(tokens[i], r)):
            if p >= 0:
                ancestors[row + j] = ancestors[row + p]
                positions[row + j] = positions[row + p] + 1
            else:
                positions[row + j] = contexts[i]
            ancestors[row + j, j // 32] |= np.uint32(1 << (j % 32))
        row += tokens[i]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=dev, dtype=torch.float32) * std).to(dt)

    up = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    return {"q": normal(n, H * hd, std=1.5), "k": normal(num_pages, G, pt, hd), "v": normal(num_pages, G, pt, hd), "table": up(table),
            "requests": up(requests), "ancestors": up(ancestors.view(np.int32)), "positions": up(positions),
            "sinks": torch.randn(H, generator=g, device=dev) if case["sink"] else None, "most_tokens": most_tokens, "most_keys": most_keys,
            "all_keys": sum(contexts) + n}


def _prepare_keep(case, seed):
    dev, dt = "cuda", getattr(torch, case["dtype"])
    r = random.Random(seed)
    R, G, hd, pt, n = case["requests"], case["groups"], case["dim"], case["page"], case["tokens"]
    per = -(-(pt + n) // pt) + 1            # pages of a request: the one that its tree begins in and those behind
    num_pages = R * per
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    cache = torch.randn((LAYERS, 2, num_pages, G, pt, hd), generator=g, device=dev, dtype=dt)
    order = np.random.RandomState(seed % (1 << 32)).permutation(num_pages).astype(np.int32).reshape(R, per)
    paths = np.full((R, 2 + case["most"]), -1, dtype=np.int32)
    for i in range(R):
        # the most probable tokens come first in a tree, so a path follows its first rows for a while and then leaves them
        kept = r.randint(1, case["most"])
        straight = r.randint(1, kept)
        paths[i, 0], paths[i, 1] = i, r.randrange(pt)
        paths[i, 2:2 + kept] = list(range(straight)) + sorted(r.sample(range(case["most"], n), kept - straight))
    block_table = torch.from_numpy(order).to(dev)
    # (address, heads, bytes a row, address of the block table) of every cache tensor: what an engine makes once
    table = torch.tensor([[cache[l, c].data_ptr(), G, hd * cache.element_size(), block_table.data_ptr()] for l in range(LAYERS) for c in range(2)],
                         dtype=torch.int64).to(dev)
    return {"cache": cache, "block_table": block_table, "paths": torch.from_numpy(paths).to(dev), "table": table}


def _prepare_copy(case, seed):
    dev = "cuda"
    r = random.Random(seed)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    arrays = torch.randint(-2 ** 31, 2 ** 31 - 1, (case["arrays"], case["blocks"], case["pieces"], case["rows"], case["row_bytes"] // 4),
                           generator=g, device=dev, dtype=torch.int32)
    m = case["moves"]
    blocks = r.sample(range(case["blocks"]), min(case["blocks"], 2 * m))
    to, sources = blocks[:m], blocks[m:]
    moves = np.zeros((m, 3), dtype=np.int32)
    for i in range(m):
        moves[i] = (r.choice(sources), to[i], case["rows"] if case["whole"] else r.randint(1, case["rows"]))
    # (address, blocks, pieces a block, bytes a piece, bytes a row) of every array: what an engine makes once
    table = torch.tensor([[arrays[a].data_ptr(), case["blocks"], case["pieces"], case["rows"] * case["row_bytes"], case["row_bytes"]]
                          for a in range(case["arrays"])], dtype=torch.int64).to(dev)
    return {"arrays": arrays, "moves": torch.from_numpy(moves).to(dev), "table": table}


def _prepare_beam(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows = case["prompts"] * case["beams"]
    logits = torch.randn((rows, case["vocab"]), generator=g, device=dev) * 2.5
    # a sharp head, as a trained model's: a few tokens far above the rest
    sharp = torch.randint(0, case["vocab"], (rows, 12), generator=g, device=dev)
    logits.scatter_(1, sharp, torch.randn((rows, 12), generator=g, device=dev) * 2.0 + 14.0)
    scores = -torch.rand((case["prompts"], case["beams"]), generator=g, device=dev) * 8.0
    if case["first"]:                       # the first step: all beams but one are not there yet
        scores[:, 1:] = -math.inf
    return {"logits": logits, "scores": scores.reshape(-1).contiguous()}


def prepare(case, seed):
    state = {"tree": _prepare_tree, "keep": _prepare_keep, "copy": _prepare_copy, "beam": _prepare_beam}[case["kind"]](case, seed)
    state["case"] = case
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------


def _plain_tree(s):
    c = s["case"]
    H, G, hd, pt, T, S = c["heads"], c["groups"], c["dim"], c["page"], s["most_tokens"], s["most_keys"]
    slot, first, count, context = (s["requests"][:, i].long() for i in range(4))
    R, n = slot.shape[0], s["q"].shape[0]
    j = torch.arange(S, device="cuda")
    i = torch.arange(T, device="cuda")
    page = s["table"][slot][:, j // pt].long().clamp(min=0)
    k = s["k"][page, :, j % pt].float()                                        # [R, S, G, hd]
    v = s["v"][page, :, j % pt].float()
    row = (first[:, None] + i).clamp(max=n - 1)                                # [R, T]
    q = s["q"][row].float().view(R, T, G, H // G, hd)
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(R, G, (H // G) * T, hd), k.permute(0, 2, 3, 1)).view(R, G, H // G, T, S)
    score = score / math.sqrt(hd)
    if c["cap"] > 0:
        score = c["cap"] * torch.tanh(score / c["cap"])
    drafted = j - context[:, None]                                             # [R, S]: a key's place in the tree, below 0 in the context
    there = drafted.clamp(0, T - 1)
    word = torch.gather(s["ancestors"][row], 2, (there // 32)[:, None, :].expand(R, T, S))
    ancestor = ((word >> (there % 32)[:, None, :].int()) & 1).bool()
    see = torch.where(drafted[:, None, :] < 0, torch.ones_like(ancestor), ancestor & (drafted < count[:, None])[:, None, :])
    if c["window"] > 0:
        place = torch.where(drafted < 0, j, s["positions"][(first[:, None] + there).clamp(max=n - 1)].long())
        see = see & (place[:, None, :] > s["positions"][row].long()[:, :, None] - c["window"])
    score = torch.where(see[:, None, None], score, torch.full((), -math.inf, device="cuda"))
    top = score.amax(-1, keepdim=True)
    if c["sink"]:
        top = torch.maximum(top, s["sinks"].view(1, G, H // G, 1, 1))
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + torch.exp(s["sinks"].view(1, G, H // G, 1, 1) - top)
    o = torch.matmul(p.view(R, G, (H // G) * T, S), v.transpose(1, 2)).view(R, G, H // G, T, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    out = torch.zeros_like(s["q"])
    real = i < count[:, None]
    out[row[real]] = o.permute(0, 3, 1, 2, 4).reshape(R, T, H * hd)[real].to(out.dtype)
    return out


def _plain_keep(s):
    pt, paths, bt = s["case"]["page"], s["paths"].long(), s["block_table"].long()
    kept = paths[:, 2:]
    real = kept >= 0
    slot, first = paths[:, :1].expand_as(kept)[real], paths[:, 1:2]
    source = (first + kept)[real]
    target = (first + torch.arange(kept.shape[1], device="cuda")).expand_as(kept)[real]
    cache = s["cache"]
    cache[:, :, bt[slot, target // pt], :, target % pt] = cache[:, :, bt[slot, source // pt], :, source % pt]
    return cache


def _plain_copy(s):
    arrays, moves = s["arrays"], s["moves"].long()
    some = torch.arange(arrays.shape[3], device="cuda") < moves[:, 2:]                          # [m, rows]
    old, new = arrays[:, moves[:, 1]], arrays[:, moves[:, 0]]
    arrays[:, moves[:, 1]] = torch.where(some[None, :, None, :, None], new, old)
    return arrays


def _plain_beam(s):
    c = s["case"]
    x = s["logits"].double()
    x = torch.where(torch.isfinite(x), x, torch.full((), -math.inf, device="cuda", dtype=torch.float64))
    top = x.amax(1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = (x - total + s["scores"].double()[:, None]).view(c["prompts"], c["beams"] * c["vocab"])
    score = torch.where(torch.isnan(score), torch.full((), -math.inf, device="cuda", dtype=torch.float64), score)
    best, at = torch.sort(score, dim=1, descending=True, stable=True)                           # of equal scores the first
    best, at = best[:, :c["choices"]], at[:, :c["choices"]]
    return best.float(), (at // c["vocab"]).int(), (at % c["vocab"]).int()


def run(s):
    c = s["case"]
    if not own:
        return {"tree": _plain_tree, "keep": _plain_keep, "copy": _plain_copy, "beam": _plain_beam}[c["kind"]](s)
    from hk_b200.csrc import ops
    if c["kind"] == "tree":
        out = torch.empty_like(s["q"])
        ops.tree_attention(s["q"], s["k"], s["v"], s["table"], s["requests"], s["ancestors"], s["positions"], out, c["heads"], c["groups"],
                           c["dim"], c["page"], c["window"], 1.0 / math.sqrt(c["dim"]), s["most_tokens"], s["most_keys"],
                           all_keys=s["all_keys"], sink=c["sink"], sinks=s["sinks"], softcap=c["cap"])
        return out
    if c["kind"] == "keep":
        ops.compact_rows(s["table"], s["paths"], s["block_table"].shape[0], s["block_table"].shape[1], c["page"], c["groups"],
                         c["dim"] * s["cache"].element_size(), s["cache"].shape[2])
        return s["cache"]
    if c["kind"] == "copy":
        ops.copy_blocks(s["table"], s["moves"], c["pieces"] * c["rows"] * c["row_bytes"])
        return s["arrays"]
    scores = torch.empty((c["prompts"], c["choices"]), dtype=torch.float32, device="cuda")
    beams, tokens = (torch.empty((c["prompts"], c["choices"]), dtype=torch.int32, device="cuda") for _ in range(2))
    ops.beam_select(s["logits"], s["scores"], c["beams"], scores, beams, tokens)
    return scores, beams, tokens


# ---- what a pass cannot do without ------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "tree":
        size = 4 if case["dtype"] == "float32" else 2
        contexts, tokens = _lengths(case)
        seen = [min(c, case["window"] - 1) if case["window"] > 0 else c for c in contexts]
        width = case["groups"] * case["dim"]
        rows = sum(tokens) * case["heads"] * case["dim"]
        return {"bytes": 2 * size * width * (sum(seen) + sum(tokens)) + 2 * size * rows,
                "flops": sum(4 * t * case["heads"] * case["dim"] * (c + t / 2) for c, t in zip(seen, tokens))}
    if case["kind"] == "keep":
        size = 4 if case["dtype"] == "float32" else 2
        # half of the longest path on average, half of that past the part which stays where it is
        moved = case["requests"] * max(1.0, case["most"] / 4)
        return {"bytes": 2 * moved * 2 * LAYERS * case["groups"] * case["dim"] * size, "flops": 0}
    if case["kind"] == "copy":
        part = 1.0 if case["whole"] else (1 + case["rows"]) / (2 * case["rows"])
        return {"bytes": 2 * case["moves"] * case["arrays"] * case["pieces"] * case["rows"] * case["row_bytes"] * part, "flops": 0}
    cells = case["prompts"] * (1 if case["first"] else case["beams"]) * case["vocab"]
    return {"bytes": 4 * cells + 12 * case["prompts"] * case["choices"], "flops": 4 * cells}


# ---- the definitions in 64 bits, apart from the plain forms -------------------------------------------------------------


def _exact_tree(case, s):
    H, G, hd, pt = case["heads"], case["groups"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    anc = s["ancestors"].cpu().numpy().view(np.uint32)
    positions = s["positions"].cpu().numpy().astype(np.int64)
    for slot, first, count, context in s["requests"].tolist():
        keys = context + count
        pages = s["table"][slot, :-(-keys // pt)].long()
        K = s["k"][pages].transpose(0, 1).reshape(G, -1, hd)[:, :keys].double()
        V = s["v"][pages].transpose(0, 1).reshape(G, -1, hd)[:, :keys].double()
        bits = np.unpackbits(anc[first:first + count].view(np.uint8), axis=1, bitorder="little")[:, :count].astype(bool)
        see = np.concatenate([np.ones((count, context), dtype=bool), bits], axis=1)
        if case["window"] > 0:
            mine = positions[first:first + count]
            back = mine[:, None] - np.concatenate([np.arange(context), mine])[None, :]
            see &= back < case["window"]
        hidden = torch.from_numpy(~see).to("cuda")
        for h in range(H):
            q = s["q"][first:first + count, h * hd:(h + 1) * hd].double()
            x = q @ K[h // (H // G)].T * hd ** -0.5
            if case["cap"] > 0:
                x = case["cap"] * torch.tanh(x / case["cap"])
            x = x.masked_fill(hidden, -math.inf)
            if case["sink"]:
                x = torch.cat([x, s["sinks"][h].double().expand(count, 1)], dim=1)
            x = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
            out[first:first + count, h * hd:(h + 1) * hd] = x[:, :keys] @ V[h // (H // G)]
    return out


def _exact_beam(case, s):
    B, K = case["prompts"], case["beams"]
    scores = s["scores"].double().view(B, K)
    out = torch.empty((B, case["choices"]), dtype=torch.float64, device="cuda")
    for b in range(B):
        rows = s["logits"][b * K:(b + 1) * K].double()
        every = rows - torch.logsumexp(rows, dim=1, keepdim=True) + scores[b][:, None]
        out[b] = torch.topk(every.reshape(-1), case["choices"]).values
    return out, None, None


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tree":
        return _exact_tree(case, s)
    if case["kind"] == "beam":
        return _exact_beam(case, s)
    if case["kind"] == "keep":
        cache, was = s["cache"], s["cache"].clone()
        pages = s["block_table"].tolist()
        for slot, first, *kept in s["paths"].tolist():
            for to, row in enumerate(r for r in kept if r >= 0):
                cache[:, :, pages[slot][(first + to) // case["page"]], :, (first + to) % case["page"]] = \
                    was[:, :, pages[slot][(first + row) // case["page"]], :, (first + row) % case["page"]]
        return cache
    arrays, was = s["arrays"], s["arrays"].clone()
    for source, target, rows in s["moves"].tolist():
        arrays[:, target, :, :rows] = was[:, source, :, :rows]
    return arrays
