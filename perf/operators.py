"""The paged K/V cache and the attention that reads it, as cases to measure: page management (fork, compact), rotary embedding
with the store into pages, attention over packed prompts, and attention of one new token per sequence, with or without a
prefix that the whole batch shares.

`run` computes an operator in plain torch, or -- where `own` is true -- through nihilus_b200.  Layouts:
  k, v   [layers][pages][kv_heads][page_tokens][head_dim] f16 or bf16      table [sequences][pages of a sequence] int32, -1 = none
  lens   [sequences] int32 tokens        refs [pages] int32, 0 = free      rows  f32 [tokens][heads * head_dim]
"""
import math
import random

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_lib = {}


def _ctx():
    """The library's context, on torch's current stream (one per process, as a program keeps it)."""
    if "ctx" not in _lib:
        from nihilus_b200 import capi

        _lib["capi"] = capi
        _lib["ctx"] = capi.Context(0)
    _lib["ctx"].use_torch_stream()
    return _lib["ctx"]


# ---- cases ----


def listed():
    llama = {"heads": 32, "kv_heads": 8, "head_dim": 128}
    small = {"heads": 32, "kv_heads": 8, "head_dim": 64}
    return [
        # four drafts off one prompt of a small model: one page each to copy, so this is the call's latency
        {"name": "fork 4 drafts", "op": "fork", "layers": 16, "kv_heads": 8, "head_dim": 64, "page": 16, "type": "f16", "parents": 1, "children": 4, "tokens": 333, "lengths": 1},
        # parallel samples of several prompts of the 8B model: 24 partly filled pages of 32 layers
        {"name": "fork 24 samples of 6", "op": "fork", "layers": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "f16", "parents": 6, "children": 24, "tokens": 1021, "lengths": 2},
        # a few short sequences leave and come back; their pages are few and small
        {"name": "compact after 3 of 9", "op": "compact", "layers": 16, "kv_heads": 8, "head_dim": 64, "page": 16, "type": "bf16", "stay": 6, "leave": 3, "tokens": 75, "lengths": 3},
        # half of a batch of the 8B model leaves: tens of pages of 8 MB move
        {"name": "compact after 8 of 16", "op": "compact", "layers": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "f16", "stay": 8, "leave": 8, "tokens": 380, "lengths": 4},
        # one decode step of a batch: one row per sequence, far positions
        {"name": "append 64 rows", "op": "append", **llama, "page": 64, "type": "f16", "sequences": 64, "new": 1, "cached": 9000, "style": "pairs", "factors": True, "lengths": 5},
        # a batch of prompts behind the q/k/v projections
        {"name": "append 4 prompts", "op": "append", **llama, "page": 64, "type": "f16", "sequences": 4, "new": 1536, "cached": 100, "style": "pairs", "factors": True, "lengths": 6},
        # one short prompt: the time to the first token of a chat line
        {"name": "prompt 77", "op": "prompt", **llama, "page": 64, "type": "f16", "sequences": 1, "new": 77, "cached": 0, "lengths": 7},
        # prompts of very different lengths in one packed call, some of them the next chunk of a longer one
        {"name": "prompt packed 11", "op": "prompt", **small, "page": 16, "type": "bf16", "sequences": 11, "new": 1300, "cached": 700, "lengths": 8},
        # one long document
        {"name": "prompt 8192", "op": "prompt", **llama, "page": 64, "type": "f16", "sequences": 1, "new": 8192, "cached": 0, "lengths": 9},
        # one user's next token
        {"name": "decode 1 x 1000", "op": "decode", **llama, "page": 64, "type": "f16", "sequences": 1, "shared": 0, "tokens": 1000, "lengths": 10},
        # a full batch of independent conversations
        {"name": "decode 48 ragged", "op": "decode", **llama, "page": 64, "type": "f16", "sequences": 48, "shared": 0, "tokens": 16001, "lengths": 11},
        # many answers behind one system prompt: its pages are read once for all
        {"name": "decode 64 shared 12288", "op": "decode", **llama, "page": 32, "type": "bf16", "sequences": 64, "shared": 12288, "tokens": 700, "lengths": 12},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(("fork", "compact", "append", "prompt", "prompt", "decode", "decode"))
    dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    c = {"op": op, "kv_heads": kv_heads, "head_dim": dim, "page": rng.choice((16, 32, 64, 128)), "type": rng.choice(("f16", "bf16")), "lengths": rng.randrange(1 << 20)}
    if op in ("fork", "compact"):
        c["layers"] = _log(rng, 1, 32)
        c["tokens"] = _log(rng, 1, 600)
        if op == "fork":
            c["parents"] = _log(rng, 1, 6)
            c["children"] = _log(rng, 1, 24)
        else:
            c["stay"], c["leave"] = _log(rng, 1, 8), _log(rng, 1, 8)
            c["tokens"] = min(c["tokens"], 380)
        return c
    c["heads"] = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
    if op == "append":
        c["sequences"] = _log(rng, 1, 64)
        c["new"] = 1 if rng.random() < 0.4 else _log(rng, 1, 4 * 1536 // c["sequences"])
        c["cached"] = rng.choice((0, _log(rng, 1, 9000)))
        c["cached"] = min(c["cached"], 4 * 9000 * 8 // (c["sequences"] * kv_heads))
        c["style"] = rng.choice(("pairs", "halves"))
        c["factors"] = rng.random() < 0.5
        c["heads"] = min(c["heads"], 32 // kv_heads * kv_heads)
    elif op == "prompt":
        c["new"] = _log(rng, 1, 4096)
        c["cached"] = rng.choice((0, _log(rng, 1, 2000)))
        most = (1 << 31) // (c["heads"] * c["new"] * (c["new"] + c["cached"]))
        c["sequences"] = _log(rng, 1, max(1, min(32, most)))
    else:
        c["sequences"] = _log(rng, 1, 96)
        c["shared"] = rng.choice((0, 0, _log(rng, 1, 16000)))
        most = 48 * 16001 * 8 // (c["sequences"] * kv_heads) - c["shared"]
        c["tokens"] = _log(rng, 1, max(1, min(16001, most // 2)))
    return c


def _lengths(case):
    """What the case's lengths are: by its own number, so that they are the same whatever the inputs' seed.
    fork: parents' tokens and each child's parent; compact: tokens of those that stay, of one half and of the other half of those that leave;
    append, prompt: (tokens before the call, new tokens) of each sequence; decode: tokens of each sequence behind the shared ones."""
    r = random.Random(case["lengths"])
    if case["op"] == "fork":
        tokens = [r.randint((case["tokens"] + 1) // 2, case["tokens"]) for _ in range(case["parents"])]
        return tokens, [i % case["parents"] for i in range(case["children"])]
    if case["op"] == "compact":
        some = lambda n: [r.randint((case["tokens"] + 1) // 2, case["tokens"]) for _ in range(n)]  # noqa: E731
        return some(case["stay"]), some((case["leave"] + 1) // 2), some(case["leave"] // 2)
    n = case["sequences"]
    if case["op"] == "decode":
        return [case["tokens"]] if n == 1 else [case["tokens"]] + [r.randint(1, case["tokens"]) for _ in range(n - 1)]
    before = [r.randint(0, case["cached"]) for _ in range(n)]
    if case["new"] == 1 or n == 1:
        return list(zip(before, [case["new"]] * n))
    return list(zip(before, [case["new"]] + [r.randint(1, case["new"]) for _ in range(n - 1)]))


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    d, kv, page = case["head_dim"], case["kv_heads"], case["page"]
    token = 2 * kv * d * 2  # bytes of one token's k and v in one layer
    if case["op"] == "fork":
        tokens, parent = _lengths(case)
        rows = sum(tokens[p] % page for p in parent)
        entries = sum(_pages(tokens[p], page) for p in parent)
        return {"bytes": 2 * rows * token * case["layers"] + 3 * 4 * entries, "flops": 0}
    if case["op"] == "compact":
        _, a, b = (sum(_pages(t, page) for t in part) for part in _lengths(case))
        return {"bytes": 2 * 2 * min(a, b) * page * token * case["layers"] + 2 * 3 * 4 * (a + b), "flops": 0}
    if case["op"] == "append":
        n = sum(new for _, new in _lengths(case))
        return {"bytes": n * (2 * 4 * case["heads"] * d + 2 * 4 * kv * d + token), "flops": 3 * n * (case["heads"] + kv) * d}
    if case["op"] == "prompt":
        lens = _lengths(case)
        pairs = sum(new * before + new * (new + 1) // 2 for before, new in lens)
        rows, keys = sum(new for _, new in lens), sum(before + new for before, new in lens)
        return {"bytes": 2 * 4 * rows * case["heads"] * d + keys * token, "flops": 4 * pairs * case["heads"] * d}
    tail = _lengths(case)
    pairs = sum(tail) + case["shared"] * len(tail)
    return {"bytes": 2 * 4 * len(tail) * case["heads"] * d + (sum(tail) + case["shared"]) * token, "flops": 4 * pairs * case["heads"] * d}


# ---- inputs ----


def _normal(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _pool(case, layers, pages, gen):
    shape = (layers, pages, case["kv_heads"], case["page"], case["head_dim"])
    return _normal(shape, gen, _TYPES[case["type"]]), _normal(shape, gen, _TYPES[case["type"]])


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(owned, most, pages, slots):
    """table, lens of pages and refs for `owned`: the pages of each sequence, in order."""
    table = [p + [-1] * (most - len(p)) for p in owned] + [[-1] * most for _ in range(slots - len(owned))]
    refs = [0] * pages
    for p in owned:
        for q in p:
            refs[q] += 1
    return _int(table), _int(refs)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    shuffle = random.Random(seed)
    page = case["page"]
    s = {"case": dict(case)}
    if case["op"] == "fork":
        tokens, parent = _lengths(case)
        held = [_pages(t, page) for t in tokens]
        pages = sum(held) + case["children"] + 5
        order = shuffle.sample(range(pages), pages)
        at = [sum(held[:i]) for i in range(len(held) + 1)]
        slots = len(tokens) + len(parent)
        s["table"], s["refs"] = _tables([order[at[i] : at[i + 1]] for i in range(len(held))], max(held) + 1, pages, slots)
        s["lens"] = _int(tokens + [0] * len(parent))
        s["parents"], s["children"] = _int(parent), _int(list(range(len(tokens), slots)))
        s["k"], s["v"] = _pool(case, case["layers"], pages, gen)
    elif case["op"] == "compact":
        parts = _lengths(case)
        tokens = [t for part in parts for t in part]
        held = [_pages(t, page) for t in tokens]
        at = [sum(held[:i]) for i in range(len(held) + 1)]
        pages = at[-1] + 3
        s["table"], s["refs"] = _tables([list(range(at[i], at[i + 1])) for i in range(len(held))], max(held), pages, len(tokens))
        s["lens"] = _int(tokens)
        first = len(parts[0])
        s["leave"] = []
        for part in parts[1:]:
            if part:
                cu = [sum(part[:i]) for i in range(len(part) + 1)]
                s["leave"].append((_int(list(range(first, first + len(part)))), _int(cu)))
                first += len(part)
        s["live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["k"], s["v"] = _pool(case, case["layers"], pages, gen)
    else:
        n, d = case["sequences"], case["head_dim"]
        lens = _lengths(case)
        shared = case.get("shared", 0)
        common = shared // page if n > 1 else 0  # whole pages that every sequence has
        total = [shared + t for t in lens] if case["op"] == "decode" else [a + b for a, b in lens]
        new = [1] * n if case["op"] == "decode" else [b for _, b in lens]
        held = [_pages(t, page) - common for t in total]
        pages = common + sum(held) + 2
        order = shuffle.sample(range(pages), pages)
        at = [common + sum(held[:i]) for i in range(n + 1)]
        s["table"], s["refs"] = _tables([order[:common] + order[at[i] : at[i + 1]] for i in range(n)], common + max(held), pages, n)
        s["lens"], s["seqs"] = _int(total), _int(shuffle.sample(range(n), n))
        names = s["seqs"].tolist()
        cu = [sum(new[i] for i in names[:k]) for k in range(n + 1)]
        s["cu"] = _int(cu) if case["op"] != "decode" else None
        s["rows"], s["most_new"], s["most"] = cu[-1], max(new), max(total)
        s["layer"] = 1 if case["op"] == "append" else 0
        s["shared"] = shared if n > 1 else 0
        s["k"], s["v"] = _pool(case, s["layer"] + 1, pages, gen)
        # queries a little stronger than unit normal: scores spread over a few units, as trained heads' do
        s["q"] = _normal((s["rows"], case["heads"] * d), gen, torch.float32, 1.5)
        s["scale"] = 1.0 / math.sqrt(d)
        if case["op"] == "append":
            s["new_k"] = _normal((s["rows"], case["kv_heads"] * d), gen, torch.float32)
            s["new_v"] = _normal((s["rows"], case["kv_heads"] * d), gen, torch.float32)
            s["base"], s["style"] = 500000.0, case["style"]
            # the long-context correction that a model file carries: low frequencies are stretched
            s["factors"] = torch.linspace(1.0, 8.0, d // 2, device="cuda") if case["factors"] else None
    s["out"] = torch.zeros_like(s["q"]) if "q" in s else None
    if own:
        _ctx()
        s["cache"] = _lib["capi"].KvCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
        if case["op"] == "append":
            s["rope"] = _lib["capi"].Rope(base=s["base"], style=s["style"], factors=s["factors"])
    return s


# ---- plain forms ----


def _free_pages(s):
    return (s["refs"] == 0).nonzero().flatten()


def _plain_free(s, seqs):
    seqs = seqs.long()
    pages = s["table"][seqs]
    held = (pages >= 0).int()
    s["refs"].index_add_(0, pages.clamp(min=0).flatten().long(), -held.flatten())
    s["table"][seqs] = -1
    s["lens"][seqs] = 0


def _plain_reserve(s, seqs, cu):
    seqs, page = seqs.long(), s["case"]["page"]
    old = s["lens"][seqs].long()
    new = old + (cu[1:] - cu[:-1]).long()
    first, last = (old + page - 1) // page, (new + page - 1) // page
    column = torch.arange(s["table"].shape[1], device="cuda")
    wanted = (column >= first[:, None]) & (column < last[:, None])
    number = wanted.flatten().cumsum(0).reshape(wanted.shape) - 1
    free = _free_pages(s)
    s["table"][seqs] = torch.where(wanted, free[number.clamp(0, free.numel() - 1)].int(), s["table"][seqs])
    taken = free[: int(wanted.sum())]
    s["refs"][taken] = 1
    s["lens"][seqs] = new.int()


def _plain_fork(s, parents, children):
    parents, children, page = parents.long(), children.long(), s["case"]["page"]
    tokens = s["lens"][parents].long()
    whole, rest = tokens // page, tokens % page
    rows = s["table"][parents]
    column = torch.arange(rows.shape[1], device="cuda")
    kept = column < whole[:, None]
    s["refs"].index_add_(0, rows.clamp(min=0).flatten().long(), kept.flatten().int())
    part = rest > 0
    number = part.long().cumsum(0) - 1
    free = _free_pages(s)
    target = free[number.clamp(min=0)]
    own_page = part[:, None] & (column == whole[:, None])
    source = (rows * own_page).sum(1).long()
    s["table"][children] = torch.where(kept, rows, torch.where(own_page, target[:, None].int(), torch.full_like(rows, -1)))
    s["lens"][children] = tokens.int()
    s["refs"][target[part]] = 1
    row = torch.arange(page, device="cuda")
    for name in ("k", "v"):
        pool = s[name]
        copied = (row < rest[part][:, None])[None, :, None, :, None]
        pool[:, target[part]] = torch.where(copied, pool[:, source[part]], pool[:, target[part]])


def _plain_compact(s):
    used = s["refs"] > 0
    live = used.sum()
    page = torch.arange(used.numel(), device="cuda")
    source, target = (used & (page >= live)).nonzero().flatten(), (~used & (page < live)).nonzero().flatten()
    for name in ("k", "v"):
        s[name][:, target] = s[name][:, source]
    moved = page.int()
    moved[source] = target.int()
    s["table"].copy_(torch.where(s["table"] >= 0, moved[s["table"].clamp(min=0).long()], s["table"]))
    s["refs"][target] = s["refs"][source]
    s["refs"][source] = 0
    s["live"][0] = live.int()


def _places(s):
    """For each row of a packed call: its sequence and its position there."""
    row = torch.arange(s["rows"], device="cuda")
    which = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    seq = s["seqs"].long()[which]
    new = (s["cu"][1:] - s["cu"][:-1]).long()[which]
    return which, seq, s["lens"][seq].long() - new + row - s["cu"].long()[which], row - s["cu"].long()[which]


def _rotate(x, position, s, heads):
    d = s["case"]["head_dim"]
    pair = torch.arange(d // 2, device="cuda", dtype=torch.float64)
    turn = s["base"] ** (-2.0 * pair / d)
    if s["factors"] is not None:
        turn = turn / s["factors"].double()
    angle = position.double()[:, None, None] * turn
    cos, sin = angle.cos().float(), angle.sin().float()
    x = x.reshape(-1, heads, d)
    x = x.reshape(-1, heads, d // 2, 2) if s["style"] == "pairs" else x.reshape(-1, heads, 2, d // 2).transpose(2, 3)
    a, b = x[..., 0], x[..., 1]
    y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1)
    return (y if s["style"] == "pairs" else y.transpose(2, 3)).reshape(-1, heads * d)


def _plain_append(s):
    c = s["case"]
    _, seq, position, _ = _places(s)
    page, slot = s["table"][seq, position // c["page"]].long(), position % c["page"]
    k = _rotate(s["new_k"], position, s, c["kv_heads"]).reshape(-1, c["kv_heads"], c["head_dim"])
    s["k"][s["layer"]][page, :, slot] = k.to(s["k"].dtype)
    s["v"][s["layer"]][page, :, slot] = s["new_v"].reshape(k.shape).to(s["v"].dtype)
    return _rotate(s["q"], position, s, c["heads"])


def _plain_attention(s):
    c = s["case"]
    n, kv, d, group = c["sequences"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    seqs = s["seqs"].long()
    pages = s["table"][seqs].long().clamp(min=0)
    gather = lambda pool: pool[s["layer"]][pages].transpose(2, 3).reshape(n, -1, kv, d).transpose(1, 2).float()  # noqa: E731
    keys = torch.arange(pages.shape[1] * c["page"], device="cuda")
    lens = s["lens"][seqs].long()
    k, v = gather(s["k"]), gather(s["v"])
    v = torch.where((keys < lens[:, None])[:, None, :, None], v, torch.zeros((), device="cuda"))
    if s["cu"] is None:
        which, index = torch.arange(n, device="cuda"), torch.zeros(n, device="cuda", dtype=torch.long)
        limit = lens[:, None] - 1
    else:
        which, _, position, index = _places(s)
        limit = torch.full((n, s["most_new"]), -1, device="cuda").index_put_((which, index), position)
    q = torch.zeros((n, s["most_new"], kv, group, d), device="cuda")
    q[which, index] = s["q"].reshape(-1, kv, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    score = (q @ k.transpose(2, 3)).mul_(s["scale"]).reshape(n, kv, group, s["most_new"], -1)
    score.masked_fill_((keys > limit[..., None])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1)
    out = (weight.reshape(n, kv, -1, keys.numel()) @ v).reshape(n, kv, group, s["most_new"], d) / total[..., None].clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4)[which, index].reshape(-1, c["heads"] * d)


def run(state):
    s, op = state, state["case"]["op"]
    if op == "fork":
        # the samples of the request before end, and new ones start from the same prompts
        if own:
            ctx = _ctx()
            ctx.kv_free(s["cache"], s["children"])
            ctx.kv_fork(s["cache"], s["parents"], s["children"])
        else:
            _plain_free(s, s["children"])
            _plain_fork(s, s["parents"], s["children"])
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "k": s["k"], "v": s["v"]}
    if op == "compact":
        # one half of the leaving sequences ends, the cache closes up and they come back behind the others; then the other half
        for seqs, cu in s["leave"]:
            if own:
                ctx = _ctx()
                ctx.kv_free(s["cache"], seqs)
                ctx.kv_compact(s["cache"], s["live"])
                ctx.kv_reserve(s["cache"], seqs, cu)
            else:
                _plain_free(s, seqs)
                _plain_compact(s)
                _plain_reserve(s, seqs, cu)
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "live": s["live"], "k": s["k"], "v": s["v"]}
    if op == "append":
        if own:
            q = _ctx().rope_kv_append(s["cache"], s["layer"], s["q"], s["new_k"], s["new_v"], s["seqs"], s["cu"], s["rope"], q_out=s["out"])
        else:
            q = _plain_append(s)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "prompt":
        if own:
            return _ctx().attn_prompt(s["cache"], s["layer"], s["q"], s["seqs"], s["cu"], s["scale"], out=s["out"])
        return _plain_attention(s)
    if own:
        return _ctx().attn_decode(s["cache"], s["layer"], s["q"], s["seqs"], s["scale"], shared=s["shared"], out=s["out"])
    return _plain_attention(s)


# ---- the definitions in 64 bits, sequence by sequence ----


def _exact_pages(s, case):
    """The cache after one pass, page by page."""
    page = case["page"]
    table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()
    k, v = s["k"].double(), s["v"].double()
    if case["op"] == "fork":
        for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
            for i in range(_pages(lens[parent], page)):
                source, rows = table[parent][i], min(page, lens[parent] - i * page)
                if rows < page:
                    target = refs.index(0)
                    refs[target] = 1
                    for pool in (k, v):
                        pool[:, target, :, :rows] = pool[:, source, :, :rows]
        return {"k": k, "v": v}
    for seqs, cu in s["leave"]:
        seqs, cu = seqs.tolist(), cu.tolist()
        for q in seqs:
            for i in range(_pages(lens[q], page)):
                refs[table[q][i]] -= 1
            lens[q] = 0
        live = sum(r > 0 for r in refs)
        for source in range(live, len(refs)):
            if refs[source] > 0:
                target = refs.index(0)
                for pool in (k, v):
                    pool[:, target] = pool[:, source]
                refs[target], refs[source] = refs[source], 0
                for q in range(len(table)):
                    for i in range(_pages(lens[q], page)):
                        if table[q][i] == source:
                            table[q][i] = target
        for j, q in enumerate(seqs):
            lens[q] = cu[j + 1] - cu[j]
            for i in range(_pages(lens[q], page)):
                table[q][i] = refs.index(0)
                refs[table[q][i]] = 1
    return {"k": k, "v": v}


def _exact_rotation(x, position, s):
    """One sequence's rows [n][heads][d] in 64 bits, pair by pair of the head."""
    d = x.shape[-1]
    y = torch.empty_like(x)
    for i in range(d // 2):
        theta = position.double() * math.exp(-2.0 * i / d * math.log(s["base"]))
        if s["factors"] is not None:
            theta = theta / float(s["factors"][i])
        a, b = (2 * i, 2 * i + 1) if s["style"] == "pairs" else (i, i + d // 2)
        c, n = theta.cos()[:, None], theta.sin()[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * n, x[..., b] * c + x[..., a] * n
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("fork", "compact"):
        return {**{n: None for n in ("table", "lens", "refs")}, **_exact_pages(s, case)}
    page, d, kv, heads = case["page"], case["head_dim"], case["kv_heads"], case["heads"]
    table, lens, seqs = s["table"].tolist(), s["lens"].tolist(), s["seqs"].tolist()
    cu = s["cu"].tolist() if s["cu"] is not None else list(range(len(seqs) + 1))
    q = s["q"].double()
    out = torch.zeros_like(q)
    k_pool, v_pool = s["k"][s["layer"]], s["v"][s["layer"]]
    new_pools = (s["k"].double(), s["v"].double()) if case["op"] == "append" else None
    for j, seq in enumerate(seqs):
        a, b, held = cu[j], cu[j + 1], lens[seq]
        ids = torch.tensor(table[seq][: _pages(held, page)], device="cuda")
        at = torch.arange(held - (b - a), held, device="cuda")
        if case["op"] == "append":
            out[a:b] = _exact_rotation(q[a:b].reshape(b - a, heads, d), at, s).reshape(b - a, heads * d)
            k = _exact_rotation(s["new_k"][a:b].double().reshape(b - a, kv, d), at, s)
            new_pools[0][s["layer"]][ids[at // page], :, at % page] = k
            new_pools[1][s["layer"]][ids[at // page], :, at % page] = s["new_v"][a:b].double().reshape(b - a, kv, d)
            continue
        future = torch.arange(held, device="cuda")[None, :] > at[:, None]
        for h in range(kv):
            k, v = k_pool[ids, h].double().reshape(-1, d)[:held], v_pool[ids, h].double().reshape(-1, d)[:held]
            for g in range(heads // kv):
                column = slice((h * (heads // kv) + g) * d, (h * (heads // kv) + g + 1) * d)
                logits = torch.where(future, -math.inf, q[a:b, column] @ k.T * s["scale"])
                out[a:b, column] = torch.softmax(logits, -1) @ v
    return out if case["op"] != "append" else {"q": out, "k": new_pools[0], "v": new_pools[1]}
