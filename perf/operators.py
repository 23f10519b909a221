"""Performance cases of the attention operators and of the paged key-value cache they share, call by call.

What a program that generates text does with them: it writes the keys and values of its tokens into pages (``append``, after
``extend`` has found the pages), has a whole prompt attended to (``prompt``), has one new token of each sequence attended to its cache
(``decode``), starts several continuations of one prompt (``fork``, and the prompt's own sequence freed), and moves the live pages
together (``compact``).

``own`` true: the calls of aspen_b200.api, on device buffers.  ``own`` false: the same results by elementary torch operations in 32 bits,
rounded once at the end.  Lengths follow from the case alone (``mix`` numbers the mixture), values and the order of pages from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    gpt2 = {"heads": 12, "kv_heads": 12, "dim": 64}         # also BERT-base
    grouped = {"heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # one short sentence through an encoder layer of BERT-base: nothing but latency
        {"name": "prompt_1x37_fp32", "op": "prompt", "type": "fp32", **gpt2, "entries": 1, "longest": 37, "ragged": False, "context": 0, "masked": False, "mix": 0},
        # prefill of eight equal prompts through GPT-2 in the framework's own type
        {"name": "prompt_8x512_fp32", "op": "prompt", "type": "fp32", **gpt2, "entries": 8, "longest": 512, "ragged": False, "context": 0, "masked": True, "mix": 0},
        # prompts of every length up to GPT-2's last position, packed without padding
        {"name": "prompt_24_packed_bf16", "op": "prompt", "type": "bf16", **gpt2, "entries": 24, "longest": 1024, "ragged": True, "context": 0, "masked": True, "mix": 1},
        # long documents, four query heads to a head of keys
        {"name": "prompt_4_long_bf16", "op": "prompt", "type": "bf16", **grouped, "entries": 4, "longest": 4096, "ragged": True, "context": 0, "masked": True, "mix": 2},
        # one user, one token, a cache that is nearly full (GPT-2)
        {"name": "decode_1x1000_fp32", "op": "decode", "type": "fp32", **gpt2, "entries": 1, "longest": 1000, "ragged": False, "page": 16, "mix": 0},
        # a batch of chats at different places
        {"name": "decode_32_ragged_fp16", "op": "decode", "type": "fp16", **gpt2, "entries": 32, "longest": 1024, "ragged": True, "page": 16, "mix": 3},
        # one very long document
        {"name": "decode_1x100003_bf16", "op": "decode", "type": "bf16", **grouped, "entries": 1, "longest": 100003, "ragged": False, "page": 64, "mix": 0},
        # a full server
        {"name": "decode_64_ragged_bf16", "op": "decode", "type": "bf16", **grouped, "entries": 64, "longest": 8192, "ragged": True, "page": 32, "mix": 4},
        # one step of a batch of chats: a token each
        {"name": "append_32x1_fp16", "op": "append", "type": "fp16", **gpt2, "entries": 32, "longest": 1, "ragged": False, "held": 700, "page": 16, "mix": 5},
        # packed prompts into an empty cache
        {"name": "append_9_prompts_bf16", "op": "append", "type": "bf16", **grouped, "entries": 9, "longest": 4096, "ragged": True, "held": 0, "page": 64, "mix": 6},
        # eight continuations of each of four prompts, in all layers of GPT-2
        {"name": "fork_4x8_fp16", "op": "fork", "type": "fp16", **gpt2, "layers": 12, "entries": 4, "copies": 8, "longest": 900, "page": 16, "mix": 7},
        # a pool of 32 chats after half of them have left, in all layers of GPT-2
        {"name": "compact_32_fp16", "op": "compact", "type": "fp16", **gpt2, "layers": 12, "entries": 32, "longest": 1024, "page": 16, "mix": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    """About the least time of a pass, in us."""
    w = work(c)
    return max(w["bytes"] / 6e6, w["flops"] / (6e7 if c["type"] == "fp32" else 1e9))


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    while True:
        op = rng.choice(["prompt", "prompt", "decode", "decode", "append", "fork", "compact"])
        kv = rng.choice([1, 2, 3, 4, 8, 12])
        c = {"op": op, "type": rng.choice(["fp32", "bf16", "fp16"]), "heads": kv * rng.choice([1, 1, 2, 4, 7, 8]), "kv_heads": kv,
             "dim": rng.choice([32, 64, 64, 80, 96, 128, 128, 256]), "mix": rng.randrange(1000)}
        if op == "prompt":
            c.update(entries=_log(rng, 1, 40), longest=_log(rng, 1, 4096), ragged=rng.random() < 0.7, context=rng.choice([0, 0, _log(rng, 1, 2000)]), masked=rng.random() < 0.8)
            if c["entries"] * c["heads"] * c["longest"] * (c["longest"] + c["context"]) > 2.2e9:      # scores of the plain form
                continue
        elif op == "decode":
            c.update(entries=_log(rng, 1, 300), longest=_log(rng, 1, 100000), ragged=rng.random() < 0.7, page=rng.choice([1, 7, 16, 32, 64, 256]))
        elif op == "append":
            step = rng.random() < 0.4
            c.update(entries=_log(rng, 1, 300), longest=1 if step else _log(rng, 2, 4096), ragged=not step, held=_log(rng, 1, 900) - 1, page=rng.choice([1, 7, 16, 32, 64, 256]))
        else:
            c.update(layers=rng.choice([1, 2, 12]), entries=_log(rng, 1, 64), longest=_log(rng, 1, 2000), page=rng.choice([1, 7, 16, 32, 64, 256]))
            if op == "fork":
                c["copies"] = _log(rng, 1, 8)
        if _cost(c) <= most[op] and _room(c) <= 6e9:
            return c


def _lengths(c, what="new"):
    """Of the entries: all the longest, or spread over 1 ... longest with the longest among them."""
    n, top = c["entries"], c["longest"]
    if not c.get("ragged", True):
        return [top] * n
    r = random.Random(1000003 * c["mix"] + 8191 * n + top)
    got = [max(1, int(top * r.random())) for _ in range(n)]
    got[r.randrange(n)] = top
    return got


def _held(c):
    """Tokens in the cache before the pass."""
    if c["op"] in ("decode", "fork", "compact"):
        return _lengths(c)
    r = random.Random(77 + c["mix"])
    return [int((c["held"] + 1) * r.random()) for _ in range(c["entries"])]


def _pages(tokens, page):
    return -(-tokens // page)


def _pool(c):
    """(pages of the pool, pages of the longest sequence, sequences)"""
    held = _held(c)
    page = c["page"]
    if c["op"] == "append":
        used = sum(_pages(h + n, page) for h, n in zip(held, _lengths(c)))
        longest = max(h + n for h, n in zip(held, _lengths(c)))
        slots = c["entries"] + 3
    elif c["op"] == "fork":
        used = sum(_pages(h, page) for h in held) + c["entries"] * c["copies"]
        longest, slots = max(held), c["entries"] * (1 + c["copies"])
    else:
        used, longest, slots = sum(_pages(h, page) for h in held), max(held), c["entries"]
    return used + used // 8 + 2, _pages(longest, page) + 1, slots


def _room(c):
    """Bytes that the inputs take."""
    if c["op"] == "prompt":
        return 0
    return 2 * c.get("layers", 1) * _pool(c)[0] * c["page"] * c["kv_heads"] * c["dim"] * _BYTES[c["type"]]


def _left(c):
    """Of a pool to be compacted: which sequences stay."""
    r = random.Random(5 + c["mix"])
    return [r.random() < 0.5 for _ in range(c["entries"])]


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def _normal(shape, g, type, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(_TYPES[type])


def _starts(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).cuda()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    D, H, KV = c["dim"], c["heads"], c["kv_heads"]
    if c["op"] == "prompt":
        q_len = _lengths(c)
        kv_len = [n + c["context"] for n in q_len]
        s["q_starts"], s["kv_starts"] = _starts(q_len), _starts(kv_len)
        # queries and keys as after a projection: scores of a few units, so that some weights matter and most do not
        s["q"] = _normal((sum(q_len), H, D), g, c["type"], 1.5)
        s["k"] = _normal((sum(kv_len), KV, D), g, c["type"])
        s["v"] = _normal((sum(kv_len), KV, D), g, c["type"])
        s["out"] = torch.zeros_like(s["q"])
        s["longest"] = (max(q_len), max(kv_len))
    else:
        pages, max_pages, slots = _pool(c)
        page, layers = c["page"], c.get("layers", 1)
        held = _held(c)
        order = np.random.RandomState(seed % (1 << 32)).permutation(pages)
        table = np.full((slots, max_pages), -1, np.int32)
        lengths, refs = np.zeros(slots, np.int32), np.zeros(pages, np.int32)
        # the entries' sequences: spread over the slots of a batch that is not full, or the first ones
        at = sorted(np.random.RandomState(c["mix"]).permutation(slots)[: c["entries"]].tolist()) if c["op"] == "append" else list(range(c["entries"]))
        stays = _left(c) if c["op"] == "compact" else [True] * c["entries"]
        used = 0
        for slot, tokens, stay in zip(at, held, stays):
            n = _pages(tokens, page)
            if stay:
                table[slot, :n] = order[used: used + n]
                refs[order[used: used + n]] = 1
                lengths[slot] = tokens
            used += n
        book = torch.from_numpy(np.concatenate([refs, lengths, [0], table.reshape(-1)]).astype(np.int32)).cuda()
        # Fresh copies of the pool's state are the first thing of a pass that changes it, on either side.
        s.update(saved=book, book=book.clone(), pages=pages, max_pages=max_pages, sequences=slots)
        s["refs"], s["lengths"] = s["book"][:pages], s["book"][pages: pages + slots]
        s["status"], s["table"] = s["book"][pages + slots: pages + slots + 1], s["book"][pages + slots + 1:].view(slots, max_pages)
        shape = (layers, pages, KV, page, D)
        s["k"], s["v"] = _normal(shape, g, c["type"]), _normal(shape, g, c["type"])
        if c["op"] == "decode":
            s["q"] = _normal((c["entries"], H, D), g, c["type"], 1.5)
            s["out"] = torch.zeros_like(s["q"])
            s["most"] = max(held)
        elif c["op"] == "append":
            new = _lengths(c)
            s["slots"], s["starts"] = torch.tensor(at, dtype=torch.int32, device="cuda"), _starts(new)
            s["rows"] = sum(new)
            s["new_k"], s["new_v"] = _normal((sum(new), KV, D), g, c["type"]), _normal((sum(new), KV, D), g, c["type"])
        elif c["op"] == "fork":
            n = c["entries"]
            s["from"] = torch.arange(n, dtype=torch.int32, device="cuda").repeat_interleave(c["copies"])
            s["to"] = torch.arange(n, n * (1 + c["copies"]), dtype=torch.int32, device="cuda")
            s["originals"] = torch.arange(n, dtype=torch.int32, device="cuda")
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program keeps for its calls: the cache's description, filled-in arguments, workspaces."""
    from aspen_b200 import api
    c = s["case"]
    kind = {"fp32": api.FP32, "bf16": api.BF16, "fp16": api.FP16}[c["type"]]
    scale = 1.0 / math.sqrt(c["dim"])
    if c["op"] == "prompt":
        s["call"] = api.PromptArgs(type=kind, heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["dim"], masked=int(c["masked"]), scale=scale,
                                   sequences=c["entries"], q_rows=s["q"].shape[0], kv_rows=s["k"].shape[0], q_starts=s["q_starts"].data_ptr(),
                                   kv_starts=s["kv_starts"].data_ptr(), q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), out=s["out"].data_ptr())
        return
    cache = s["cache"] = api.Cache(type=kind, layers=c.get("layers", 1), pages=s["pages"], page_size=c["page"], kv_heads=c["kv_heads"], head_dim=c["dim"],
                                   sequences=s["sequences"], max_pages=s["max_pages"], k=s["k"].data_ptr(), v=s["v"].data_ptr(),
                                   page_table=s["table"].data_ptr(), lengths=s["lengths"].data_ptr(), refs=s["refs"].data_ptr(), status=s["status"].data_ptr())
    if c["op"] == "decode":
        need = cache.decode_workspace(c["entries"], c["heads"])
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        s["call"] = api.DecodeArgs(entries=c["entries"], heads=c["heads"], scale=scale, q=s["q"].data_ptr(), out=s["out"].data_ptr(),
                                   workspace=s["workspace"].data_ptr(), workspace_bytes=need)
    else:
        need = cache.workspace(c["entries"] * c.get("copies", 1))
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        if c["op"] == "append":
            s["call"] = api.AppendArgs(entries=c["entries"], rows=s["rows"], slots=s["slots"].data_ptr(), starts=s["starts"].data_ptr(),
                                       k=s["new_k"].data_ptr(), v=s["new_v"].data_ptr())


# ---- one pass ----------------------------------------------------------------------------------------------------------------

def run(state):
    s = state
    op = s["case"]["op"]
    if op in ("append", "fork", "compact"):
        s["book"].copy_(s["saved"])
    if own:
        from aspen_b200 import api
        stream = torch.cuda.current_stream().cuda_stream
        if op == "prompt":
            api.attention_prompt(s["call"], stream)
        elif op == "decode":
            s["cache"].decode(0, s["call"], stream)
        else:
            space = (s["workspace"].data_ptr(), s["workspace"].numel())
            if op == "append":
                s["cache"].extend(s["slots"].data_ptr(), s["starts"].data_ptr(), s["case"]["entries"], *space, stream)
                s["cache"].append(0, s["call"], stream)
            elif op == "fork":
                s["cache"].fork(s["from"].data_ptr(), s["to"].data_ptr(), s["from"].numel(), *space, stream)
                s["cache"].free(s["originals"].data_ptr(), s["originals"].numel(), stream)
            else:
                s["cache"].compact(*space, stream)
    elif op == "prompt":
        s["out"] = _plain_prompt(s)
    elif op == "decode":
        s["out"] = _plain_decode(s)
    elif op == "append":
        _plain_append(s)
    elif op == "fork":
        _plain_fork(s)
    else:
        _plain_compact(s)
    return s["out"] if op in ("prompt", "decode") else [s["k"], s["v"], s["book"]]


def _softmax_weighted(scores, seen, v):
    """softmax over the last axis of what is seen, times v; zeros where nothing is."""
    scores = scores.masked_fill(~seen, float("-inf"))
    most = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - most)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total.masked_fill(total == 0, 1)


def _plain_prompt(s):
    """Sequences side by side, padded to the longest."""
    c = s["case"]
    H, KV, D = c["heads"], c["kv_heads"], c["dim"]
    (Q, K), n = s["longest"], c["entries"]
    qs, ks = s["q_starts"].long(), s["kv_starts"].long()
    q_len, k_len = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    i, j = torch.arange(Q, device="cuda"), torch.arange(K, device="cuda")
    qi = (qs[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    kj = (ks[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][qi].float().view(n, Q, KV, H // KV, D).permute(0, 2, 3, 1, 4)
    k = s["k"][kj].float().permute(0, 2, 3, 1)[:, :, None]
    v = s["v"][kj].float().permute(0, 2, 1, 3)[:, :, None]
    seen = (j < k_len[:, None])[:, None].expand(n, Q, K)
    if c["masked"]:
        seen = seen & (j <= (i[:, None] + (k_len - q_len)[:, None, None]))
    scores = torch.matmul(q, k) * (1.0 / math.sqrt(D))
    out = _softmax_weighted(scores, seen[:, None, None], v).permute(0, 3, 1, 2, 4).reshape(n, Q, H, D)
    return out[i < q_len[:, None]].to(s["q"].dtype)


def _plain_decode(s):
    c = s["case"]
    H, KV, D, page, n = c["heads"], c["kv_heads"], c["dim"], c["page"], c["entries"]
    wide = _pages(s["most"], page)
    table = s["table"][:n, :wide].long().clamp(min=0)
    k = s["k"][0][table].transpose(2, 3).reshape(n, wide * page, KV, D).float().permute(0, 2, 3, 1)
    v = s["v"][0][table].transpose(2, 3).reshape(n, wide * page, KV, D).float().permute(0, 2, 1, 3)
    seen = (torch.arange(wide * page, device="cuda") < s["lengths"][:n, None])[:, None, None]
    q = s["q"].float().view(n, KV, H // KV, D)
    return _softmax_weighted(torch.matmul(q, k) * (1.0 / math.sqrt(D)), seen, v).view(n, H, D).to(s["q"].dtype)


def _plain_append(s):
    page = s["case"]["page"]
    slots, starts = s["slots"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    held = s["lengths"][slots].long()
    first = (held + page - 1) // page
    need = (held + new + page - 1) // page - first
    which = torch.repeat_interleave(torch.arange(slots.numel(), device="cuda"), need)
    pages = torch.nonzero(s["refs"] == 0).view(-1)[: which.numel()]
    at = first[which] + torch.arange(which.numel(), device="cuda") - (need.cumsum(0) - need)[which]
    s["table"][slots[which], at] = pages.int()
    s["refs"][pages] = 1
    s["lengths"][slots] = (held + new).int()
    row = torch.repeat_interleave(torch.arange(slots.numel(), device="cuda"), new, output_size=s["rows"])
    position = held[row] + torch.arange(s["rows"], device="cuda") - starts[row]
    to = s["table"][slots[row], position // page].long()
    s["k"][0][to, :, position % page] = s["new_k"]
    s["v"][0][to, :, position % page] = s["new_v"]


def _plain_fork(s):
    page = s["case"]["page"]
    a, b = s["from"].long(), s["to"].long()
    held = s["lengths"][a].long()
    full, rest = held // page, held % page
    part = torch.nonzero(rest > 0).view(-1)
    pages = torch.nonzero(s["refs"] == 0).view(-1)[: part.numel()]
    column = torch.arange(s["max_pages"], device="cuda")
    rows = torch.where(column < full[:, None], s["table"][a], -1)
    shared = rows[rows >= 0].long()
    old = s["table"][a[part], full[part]].long()
    rows[part, full[part]] = pages.int()
    s["table"][b] = rows
    s["lengths"][b] = held.int()
    s["refs"].index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    s["refs"][pages] = 1
    used = (torch.arange(page, device="cuda") < rest[part, None])[None, :, None, :, None]
    for cache in (s["k"], s["v"]):
        cache[:, pages] = torch.where(used, cache[:, old], cache[:, pages])
    gone = s["originals"].long()
    rows = s["table"][gone]
    freed = rows[rows >= 0].long()
    s["refs"].index_add_(0, freed, torch.full_like(freed, -1, dtype=torch.int32))
    s["table"][gone] = -1
    s["lengths"][gone] = 0


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    number = torch.arange(s["pages"], device="cuda")
    live = refs > 0
    count = live.sum()
    old, new = torch.nonzero(live & (number >= count)).view(-1), torch.nonzero(~live & (number < count)).view(-1)
    for cache in (s["k"], s["v"]):
        cache[:, new] = cache[:, old]
    refs[new] = refs[old]
    refs[old] = 0
    number[old] = new
    table.copy_(torch.where(table >= 0, number[table.long().clamp(min=0)].int(), -1))


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------

def work(case):
    c = case
    size, H, KV, D = _BYTES[c["type"]], c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "prompt":
        pairs = 0
        for n in _lengths(c):
            m = n + c["context"]
            pairs += n * m - n * (n - 1) // 2 if c["masked"] else n * m
        rows, keys = sum(_lengths(c)), sum(n + c["context"] for n in _lengths(c))
        return {"bytes": size * D * (2 * rows * H + 2 * keys * KV), "flops": 4 * pairs * H * D}
    held = _held(c)
    token = 2 * KV * D * size               # key and value, one layer
    if c["op"] == "decode":
        return {"bytes": sum(held) * token + 2 * c["entries"] * H * D * size + 4 * sum(_pages(h, c["page"]) for h in held), "flops": 4 * sum(held) * H * D}
    state = 4 * (_pool(c)[0] + _pool(c)[2] * (1 + _pool(c)[1]))
    if c["op"] == "append":
        return {"bytes": 2 * sum(_lengths(c)) * token + 3 * state, "flops": 0}
    if c["op"] == "fork":
        return {"bytes": 2 * c["layers"] * c["copies"] * sum(h % c["page"] for h in held) * token + 3 * state, "flops": 0}
    # what moves depends on where the live pages lie: with an even spread, this share of them lies behind the new end
    live, pages = sum(_pages(h, c["page"]) for h, stay in zip(held, _left(c)) if stay), _pool(c)[0]
    return {"bytes": 2 * c["layers"] * live * (1 - live / pages) * c["page"] * token + 3 * state, "flops": 0}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    if c["op"] not in ("prompt", "decode") or work(c)["flops"] > 1e13:
        return None
    s = prepare(c, seed)
    D, group = c["dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def attend(q, k, v, first):
        """q [n][H][D], k, v [m][KV][D]; query i sees the keys up to first + i."""
        for h in range(c["heads"]):
            for at in range(0, q.shape[0], 2048):
                a = q[at: at + 2048, h].double() / math.sqrt(D)
                m = k.shape[0] if first is None else min(k.shape[0], first + at + a.shape[0])
                if m <= 0:
                    continue
                x = a @ k[:m, h // group].double().T
                if first is not None:
                    sees = torch.arange(m, device="cuda")[None] <= first + at + torch.arange(a.shape[0], device="cuda")[:, None]
                    x = torch.where(sees, x, torch.full_like(x, -math.inf))
                w = torch.softmax(x, -1)
                yield h, at, torch.nan_to_num(w) @ v[:m, h // group].double()

    if c["op"] == "prompt":
        qs, ks = s["q_starts"].tolist(), s["kv_starts"].tolist()
        for a, b, x, y in zip(qs, qs[1:], ks, ks[1:]):
            for h, at, r in attend(s["q"][a:b], s["k"][x:y], s["v"][x:y], (y - x) - (b - a) if c["masked"] else None):
                out[a + at: a + at + r.shape[0], h] = r
    else:
        for e, n in enumerate(_held(c)):
            pages = s["table"][e, : _pages(n, c["page"])].long()
            k, v = (s[x][0][pages].permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], D)[:n] for x in ("k", "v"))
            for h, at, r in attend(s["q"][e: e + 1], k, v, None):
                out[e, h] = r[0]
    return out
