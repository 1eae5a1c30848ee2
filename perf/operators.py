"""Timed cases of exact attention over a cache of key and value rows, and of what keeps such a cache small: attention of
decoded tokens and of prompt chunks (capped scores, distance bias, window, prefix and document masks), attention of a
tree of drafted tokens, the weight that each cached row receives, and the removal of the rows that receive the least.

A cache is a run of rows a sequence, [row][kv_head][head_dim]; queries and outputs are [token][head][head_dim].
"""
import math

import torch

own = False

DEV = "cuda"
_stream = None  # the framework's calls are made on one stream of the caller's


def _attend(**more):
    case = dict(op="attend", dtype="bf16", d=128, kv_heads=8, group=4, seqs=1, rows=4096, ragged=False, tokens=1, softcap=0.0, alibi=False, window=0,
                prefix=0, documents=0, moved=False)
    case.update(more)
    return case


def listed():
    return [
        # One decoded token of a short conversation: what counts is the call itself.
        dict(_attend(rows=512), name="decode_short"),
        # One decoded token on a long context, scores capped: the cache is read once.
        dict(_attend(rows=131072, softcap=50.0), name="decode_128k_softcap"),
        # A batch of decoded tokens of a model with a distance bias; sequences of different lengths, rows kept by an earlier eviction (positions of their own).
        dict(_attend(seqs=48, rows=9001, ragged=True, alibi=True, moved=True), name="decode_batch_alibi"),
        # A packed prompt of several documents: each token sees its own document's.
        dict(_attend(rows=8192, tokens=8192, documents=9), name="prompt_documents"),
        # A chunk of a long prompt under a sliding window and a cap, as a scheduler of chunked prompts calls it.
        dict(_attend(rows=16384, tokens=2048, softcap=30.0, window=4096), name="prompt_chunk_window"),
        # float32 caches: short continuations with a shared prefix that all of them see, odd sizes.
        dict(_attend(dtype="f32", d=96, kv_heads=4, group=3, seqs=5, rows=1501, ragged=True, tokens=37, prefix=129, alibi=True), name="chunk_f32_prefix"),
        # A few drafted tokens of one sequence.
        dict(op="tree", dtype="bf16", d=128, kv_heads=8, group=4, seqs=1, rows=2003, ragged=False, tokens=7, softcap=0.0, window=0, name="tree_few"),
        # Wide trees of drafted tokens for a batch of sequences.
        dict(op="tree", dtype="bf16", d=128, kv_heads=8, group=4, seqs=16, rows=8192, ragged=True, tokens=63, softcap=0.0, window=0, name="tree_batch"),
        # After a decode step of a batch: the weight that each cached row received.
        dict(op="observe", dtype="bf16", d=128, kv_heads=8, group=4, seqs=16, rows=8192, ragged=True, tokens=1, softcap=0.0, window=0, name="observe_decode"),
        # After a prompt: the weight that its rows receive from its last 64 tokens.
        dict(op="observe", dtype="bf16", d=128, kv_heads=8, group=4, seqs=1, rows=32768, ragged=False, tokens=64, softcap=0.0, window=0, name="observe_prompt"),
        # One conversation's cache, a few rows over its budget.
        dict(op="evict", dtype="f32", d=64, kv_heads=2, seqs=1, rows=1100, ragged=False, budget=1024, sink=4, recent=64, tiles=False, name="evict_short"),
        # Prompts into caches an eighth as long, their 128-byte tiles with them.
        dict(op="evict", dtype="bf16", d=128, kv_heads=8, seqs=8, rows=32768, ragged=True, budget=4096, sink=4, recent=512, tiles=True, name="evict_prompts"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend"] * 5 + ["tree"] * 2 + ["observe"] * 2 + ["evict"] * 2)
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 4, 8])
    dtype, d = rng.choice(["bf16"] * 4 + ["f32"]), rng.choice([64, 80, 96, 128, 128, 128, 256])
    seqs, ragged = _spread(rng, 1, 64), rng.random() < 0.6
    most = (1 << 18) * 8 // kv_heads * 128 // max(d, 128) // seqs  # rows of a sequence
    if op == "evict":
        rows = min(most, _spread(rng, 65, 65536))
        budget = max(17, int(rows * rng.uniform(0.05, 0.98)))
        return dict(op=op, dtype=dtype, d=d, kv_heads=kv_heads, seqs=seqs, rows=rows, ragged=ragged, budget=budget, sink=rng.choice([0, 1, 4]),
                    recent=_spread(rng, 1, max(1, budget // 4)), tiles=rng.random() < 0.3)
    kind = dict(op=op, dtype=dtype, d=d, kv_heads=kv_heads, group=group, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), window=rng.choice([0, 0, 0, 1]) * _spread(rng, 16, 4096))
    if op == "attend":
        long = rng.random() < 0.5  # a prompt or a chunk of one, else decoded tokens
        tokens = _spread(rng, 5, 4096) if long else rng.choice([1, 1, 1, 2, 3])
        if long:
            seqs = min(seqs, 8)
            pairs = (1 << 25) if dtype == "f32" else (1 << 27)  # (head, token, row) triples stay below the largest listed case's
            tokens = max(1, min(tokens, int(math.sqrt(pairs / (seqs * kv_heads * group)))))
            rows = min(most, max(tokens, _spread(rng, tokens, max(tokens + 1, pairs // (seqs * kv_heads * group * tokens)))))
        else:
            rows = min(most, _spread(rng, tokens + 1, 131072))
        return _attend(seqs=seqs, rows=rows, ragged=ragged, tokens=tokens, alibi=rng.random() < 0.3, prefix=rng.choice([0, 0, 1]) * _spread(rng, 1, rows),
                       documents=rng.choice([0, 0, 2, 7]), moved=rng.random() < 0.3, **{k: v for k, v in kind.items() if k != "op"})
    tokens = _spread(rng, 1, 64) if op == "tree" else rng.choice([1, 1, 16, 32, 64])
    seqs = min(seqs, 16)
    rows = max(tokens, min(most, (1 << 22) // (seqs * tokens), _spread(rng, 64, 65536)))
    return dict(kind, seqs=seqs, rows=rows, ragged=ragged, tokens=tokens)


# --------------------------------------------------------------------------- inputs
def _lengths(case):
    n, low = case["rows"], max(case.get("tokens", 1), case["rows"] // 3)
    return [n - ((i * 40503 + 17) % 65536) * (n - low) // 65536 if case["ragged"] else n for i in range(case["seqs"])]


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _begins(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _documents(gen, n, count):
    """n rows in runs of `count` documents, numbered from 1."""
    cuts = torch.sort(torch.randint(0, n, (count - 1,), generator=gen, device=DEV)).values
    return (torch.bucketize(torch.arange(n, device=DEV), cuts, right=True) + 1).to(torch.int32)


def _parents(gen, tokens):
    """A tree: each drafted token's parent is one of the up to twelve before it, the first has none."""
    at = torch.arange(tokens, device=DEV)
    back = 1 + torch.randint(0, 12, (tokens,), generator=gen, device=DEV)
    return torch.where(at - back >= 0, at - back, torch.full_like(at, -1)).to(torch.int32)


def _ancestors(parents):
    """[sequence][token][token]: whether the second is the first or one of its ancestors."""
    seqs, tokens = parents.shape
    seen = torch.eye(tokens, dtype=torch.bool, device=DEV).repeat(seqs, 1, 1)
    at = parents.long()
    link = torch.zeros(seqs, tokens, tokens, device=DEV)
    link.scatter_(2, at.clamp(min=0)[:, :, None], (at >= 0).float()[:, :, None])
    reach = seen.float()
    for _ in range(max(1, math.ceil(math.log2(tokens + 1)))):  # each time twice as far up the tree
        reach = ((reach + link @ reach) > 0).float()
        link = ((link @ link) > 0).float()
    return reach > 0


def _inputs(case, seed):
    gen, lens, tokens, dtype = _gen(seed), _lengths(case), case.get("tokens", 1), _type(case)
    begins = _begins(lens)
    total, heads, d = begins[-1], case["kv_heads"], case["d"]
    chan = torch.exp(0.5 * torch.randn(d, generator=gen, device=DEV))
    st = dict(case, lens=lens, begins=begins, total=total)
    st["keys"] = (torch.randn(total, heads, d, generator=gen, device=DEV) * chan).to(dtype)
    st["values"] = torch.randn(total, heads, d, generator=gen, device=DEV).to(dtype)
    if case["op"] == "evict":
        # rows that many tokens looked at and rows that hardly one did; some never seen, which tie at zero
        w = torch.randn(heads, total, generator=gen, device=DEV).mul(2.0).exp()
        st["weights"] = torch.where(torch.rand(heads, total, generator=gen, device=DEV) < 0.1, torch.zeros_like(w), w)
        st["positions"] = torch.cat([torch.arange(n, device=DEV) * 3 // 2 for n in lens]).to(torch.int32).repeat(heads, 1)
        if case["tiles"]:
            st["rows128"] = torch.randint(0, 256, (heads, total, 128), generator=gen, device=DEV, dtype=torch.uint8)
        return st
    n_heads = heads * case["group"]
    st["n_heads"], st["n_tokens"] = n_heads, case["seqs"] * tokens
    st["q"] = (torch.randn(case["seqs"] * tokens, n_heads, d, generator=gen, device=DEV) * 1.5).to(dtype)
    if case.get("moved"):
        # rows that an eviction has left, in another order than they were written
        gaps = [torch.cumsum(torch.randint(1, 4, (n,), generator=gen, device=DEV), 0) for n in lens]
        mixed = [torch.cat([g[torch.randperm(n - tokens, generator=gen, device=DEV)], g[n - tokens:]]) for g, n in zip(gaps, lens)]
        st["positions"] = torch.cat(mixed).to(torch.int32)
        st["q_positions"] = torch.cat([g[-tokens:] for g in mixed]).to(torch.int32)
    if case.get("documents"):
        st["docs"] = torch.cat([_documents(gen, n, case["documents"]) for n in lens])
        st["q_docs"] = torch.cat([st["docs"][b - tokens:b] for b in begins[1:]])
    if case.get("alibi"):
        st["slopes"] = (2.0 ** (-8.0 * torch.arange(1, n_heads + 1, device=DEV) / n_heads)).float()
    if case.get("prefix"):
        st["prefixes"] = torch.tensor([min(case["prefix"], n) for n in lens], dtype=torch.int32, device=DEV)
    if case["op"] == "tree":
        st["parents"] = torch.cat([_parents(gen, tokens) for _ in lens])
    return st


def prepare(case, seed):
    global _stream
    st = _inputs(case, seed)
    if case["op"] == "evict":
        heads, d, seqs, budget = case["kv_heads"], case["d"], case["seqs"], case["budget"]
        room = seqs * budget
        st["to"] = dict(keys=torch.zeros(room, heads, d, dtype=_type(case), device=DEV), values=torch.zeros(room, heads, d, dtype=_type(case), device=DEV),
                        positions=torch.zeros(heads, room, dtype=torch.int32, device=DEV), weights=torch.zeros(heads, room, device=DEV),
                        source=torch.full((seqs, heads, budget), -1, dtype=torch.int32, device=DEV))
        if case["tiles"]:
            st["to"]["rows128"] = torch.zeros(heads, room, 128, dtype=torch.uint8, device=DEV)
    else:
        st["out"] = torch.empty(st["n_tokens"], st["n_heads"], case["d"], dtype=_type(case), device=DEV)
        st["lse"] = torch.empty(st["n_tokens"], st["n_heads"], device=DEV)
        if case["op"] == "observe":
            # what earlier steps left there, of the size of what this one adds
            st["weights_in"] = torch.rand(case["kv_heads"], st["total"], generator=_gen(seed + 1), device=DEV) * (case["group"] * case["tokens"] / case["rows"])
            st["weights"] = torch.empty_like(st["weights_in"])
            st["lse"] = _softmax_parts(st, _scores(st))[1].contiguous()  # (what the attention of the same step wrote)
    if own:  # the handles that a program keeps: where its cache lies, where its queries come to lie, the table of its sequences
        import slhav2_b200 as S

        if _stream is None:
            _stream = torch.cuda.Stream()
        S.set_stream(_stream.cuda_stream)
        torch.cuda.synchronize()
        dtype = S.BF16 if case["dtype"] == "bf16" else S.F32
        tokens = case.get("tokens", 0)
        st["segs"] = S.make_segments([(b, n, i * tokens, tokens, 0) for i, (b, n) in enumerate(zip(st["begins"], st["lens"]))])
        per_head = case["op"] == "evict"
        st["cache"] = S.KvCache(st["keys"], st["values"], case["kv_heads"], case["d"], dtype=dtype, positions=st.get("positions"), documents=st.get("docs"),
                                entry_head_stride=st["total"] if per_head else 0)
        if per_head:
            to, room = st["to"], case["seqs"] * case["budget"]
            st["small"] = S.KvCache(to["keys"], to["values"], case["kv_heads"], case["d"], dtype=dtype, positions=to["positions"], entry_head_stride=room)
            st["to_segs"] = S.make_segments([(i * case["budget"], case["budget"], 0, 0, 0) for i in range(case["seqs"])])
        else:
            st["queries"] = S.CacheQueries(st["q"], st["n_tokens"], st["n_heads"], case["d"], softcap=case["softcap"], window=case["window"],
                                           slopes=st.get("slopes"), prefix=st.get("prefixes"), positions=st.get("q_positions"), documents=st.get("q_docs"))
    return st


# --------------------------------------------------------------------------- plain forms
def _rows_of(st):
    """[sequence][row] places in the cache, and which of them are rows of the sequence."""
    lens, at = torch.tensor(st["lens"], device=DEV), torch.arange(max(st["lens"]), device=DEV)
    begin = torch.tensor(st["begins"][:-1], device=DEV)
    there = at < lens[:, None]
    return torch.where(there, begin[:, None] + at, 0), there


def _seen(st, where, there):
    """[sequence][token][row]: the rows that a token sees, and the distance between the two."""
    seqs, tokens = st["seqs"], st["tokens"]
    lens = torch.tensor(st["lens"], device=DEV)
    at = torch.arange(where.shape[1], device=DEV)
    if "positions" in st:
        row_pos, q_pos = st["positions"][where].long(), st["q_positions"].long().view(seqs, tokens)
    else:
        row_pos, q_pos = at.expand(seqs, -1), lens[:, None] - tokens + torch.arange(tokens, device=DEV)
    drafted = None
    if st["op"] == "tree":
        family = _ancestors(st["parents"].view(seqs, tokens))
        depth = family.sum(2) - 1
        q_pos = lens[:, None] - tokens + depth
        draft = at - (lens[:, None] - tokens)  # a row's number among the drafted ones
        of = draft.clamp(0, tokens - 1)
        drafted = draft >= 0
        row_pos = torch.where(drafted, (lens - tokens)[:, None] + depth.gather(1, of), row_pos)
    away = q_pos[:, :, None] - row_pos[:, None, :]
    seen = away >= 0
    if st["window"]:
        seen &= away < st["window"]
    if drafted is not None:
        seen &= ~drafted[:, None, :] | family.gather(2, of[:, None, :].expand(-1, tokens, -1))
    if "prefixes" in st:
        seen |= (row_pos < st["prefixes"].long()[:, None])[:, None, :]
    if "docs" in st:
        seen &= st["docs"][where][:, None, :] == st["q_docs"].view(seqs, tokens)[:, :, None]
    return seen & there[:, None, :], away


def _scores(st):
    """[sequence][kv_head][group][token][row], -inf where a row is not seen."""
    where, there = _rows_of(st)
    seen, away = _seen(st, where, there)
    seqs, tokens, heads, d = st["seqs"], st["tokens"], st["kv_heads"], st["d"]
    q = st["q"].float().view(seqs, tokens, heads, -1, d).permute(0, 2, 3, 1, 4)
    group, n = q.shape[2], where.shape[1]
    k = st["keys"][where].float().permute(0, 2, 3, 1)  # [sequence][kv_head][d][row]
    s = torch.matmul(q.reshape(seqs, heads, group * tokens, d), k).view(seqs, heads, group, tokens, n) * d ** -0.5
    del k
    if st["softcap"]:
        s = st["softcap"] * torch.tanh(s / st["softcap"])
    if "slopes" in st:
        s -= st["slopes"].view(1, heads, group, 1, 1) * away.abs().float()[:, None, None]
    return s.masked_fill_(~seen[:, None, None], -math.inf)


def _softmax_parts(st, s):
    """exp(score - largest), and the logarithm of the sums as [token][head]."""
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1)
    lse = torch.log(total) + top[..., 0]
    return p, lse.permute(0, 3, 1, 2).reshape(st["n_tokens"], st["n_heads"]), total


def _plain_attend(st):
    p, lse, total = _softmax_parts(st, _scores(st))
    where, _ = _rows_of(st)
    seqs, heads, group, tokens, n = p.shape
    v = st["values"][where].float().permute(0, 2, 1, 3)  # [sequence][kv_head][row][d]
    o = torch.matmul(p.view(seqs, heads, group * tokens, n), v).view(seqs, heads, group, tokens, -1)
    o /= torch.where(total > 0, total, 1.0)[..., None]
    st["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(st["out"].shape))
    st["lse"].copy_(lse)
    return st["out"], st["lse"]


def _plain_observe(st):
    s = _scores(st)
    seqs, heads, group, tokens, n = s.shape
    lse = st["lse"].view(seqs, tokens, heads, group).permute(0, 2, 3, 1)[..., None]
    w = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)).sum((2, 3))  # [sequence][kv_head][row]
    _, there = _rows_of(st)
    torch.mul(st["weights_in"], 0.5, out=st["weights"])
    st["weights"] += w.permute(1, 0, 2)[:, there]
    return st["weights"]


def _plain_evict(st):
    where, there = _rows_of(st)
    seqs, heads, budget, to = st["seqs"], st["kv_heads"], st["budget"], st["to"]
    head = torch.arange(heads, device=DEV)[:, None]
    pos = st["positions"][:, where].long()  # [kv_head][sequence][row]
    newest = pos.masked_fill(~there, -1).amax(2, keepdim=True)
    pinned = (pos < st["sink"]) | (newest - pos < st["recent"])
    key = torch.where(pinned, math.inf, st["weights"][:, where]).masked_fill(~there, -math.inf)
    n = key.shape[2]
    order = torch.sort(key, dim=2, descending=True, stable=True).indices
    kept = torch.zeros_like(key, dtype=torch.bool).scatter_(2, order[:, :, :budget], True) & there
    # a row that stays within the budget keeps its place; the others' places go to the kept rows behind it, in order
    short = min(budget, n)
    front = kept[:, :, :short]
    behind = torch.sort((~kept[:, :, short:]).to(torch.int8), dim=2, stable=True).indices + short
    rank = (~front).cumsum(2) - 1
    at = torch.arange(short, device=DEV)
    if n > short:
        source = torch.where(front, at, behind.gather(2, rank.clamp(0, n - short - 1)))
    else:
        source = at.expand_as(front).clone()
    valid = (at < torch.tensor(st["lens"], device=DEV)[:, None]).expand_as(front)  # [kv_head][sequence][place]
    source = torch.where(valid, source, -1)
    rows = torch.where(valid, torch.tensor(st["begins"][:-1], device=DEV)[:, None] + source.clamp(min=0), 0)
    place = (torch.arange(seqs, device=DEV)[:, None] * budget + at).expand_as(front)[valid]
    h = head[:, :, None].expand_as(front)[valid]
    r = rows[valid]
    for name in ("keys", "values"):
        to[name][place, h] = st[name][r, h]
    for name in ("positions", "weights") + (("rows128",) if st["tiles"] else ()):
        to[name][h, place] = st[name][h, r]
    to["source"][:, :, :short] = source.permute(1, 0, 2).to(torch.int32)
    return to


def run(st):
    op = st["op"]
    if own:
        import slhav2_b200 as S

        if op == "attend":
            S.attend_cache(st["cache"], st["segs"], st["queries"], st["out"], st["lse"])
            return st["out"], st["lse"]
        if op == "tree":
            S.attend_tree(st["cache"], st["segs"], st["queries"], st["parents"], st["out"], st["lse"])
            return st["out"], st["lse"]
        if op == "observe":
            S.observe_cache(st["cache"], st["segs"], st["queries"], st["lse"], st["weights"], st["total"], weights_in=st["weights_in"], decay=0.5)
            return st["weights"]
        to = st["to"]
        S.evict_cache(st["cache"], st["segs"], st["weights"], st["total"], st["budget"], sink_window=st["sink"], recent_window=st["recent"],
                      to=st["small"], to_segments=st["to_segs"], weights_to=to["weights"], weights_to_head_stride=st["seqs"] * st["budget"],
                      tiles=st.get("rows128"), tile_head_stride=st["total"], tiles_to=to.get("rows128"), tiles_to_head_stride=st["seqs"] * st["budget"],
                      source_out=to["source"])
        return to
    if op in ("attend", "tree"):
        return _plain_attend(st)
    return _plain_observe(st) if op == "observe" else _plain_evict(st)


# --------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """(token, row) pairs that are seen, about, and the rows that any token sees."""
    pairs, rows = 0.0, 0
    tokens, window, prefix = case["tokens"], case["window"], case.get("prefix", 0)
    for n in _lengths(case):
        ctx = n - tokens
        span = min(window, n) if window and not case.get("moved") else n
        seen = sum(min(ctx + t + 1, span) for t in range(tokens)) if tokens <= 4096 else tokens * (ctx + (tokens + 1) / 2)
        docs = max(1, case.get("documents", 0))
        if docs > 1:
            # a token sees its document's earlier rows: of runs cut at random, twice the share of equal ones
            seen = min(seen, tokens * 2.0 * n / (docs + 1) / 2)
        seen = max(seen, float(min(prefix, n)) * tokens / docs)
        pairs += min(seen, float(tokens) * n)
        rows += n if docs > 1 or not window else min(n, span + tokens - 1 + min(prefix, n))
    return pairs, rows


def work(case):
    e, d, heads = (2 if case["dtype"] == "bf16" else 4), case["d"], case["kv_heads"]
    if case["op"] == "evict":
        # every weight and position once; the kept rows, with what belongs to them, once and back
        rows = sum(_lengths(case))
        kept = sum(min(n, case["budget"]) for n in _lengths(case))
        each = 2 * (2 * d * e + 4 + 4 + (128 if case["tiles"] else 0)) + 4
        return {"bytes": heads * (8 * rows + each * kept), "flops": 0}
    pairs, rows = _pairs(case)
    n_q = case["seqs"] * case["tokens"] * heads * case["group"]
    flops = 2 * pairs * heads * case["group"] * d
    if case["op"] == "observe":
        return {"bytes": heads * rows * (d * e + 4) + heads * sum(_lengths(case)) * 4 + n_q * (d * e + 4), "flops": flops}
    return {"bytes": 2 * heads * rows * d * e + n_q * (2 * d * e + 4) + rows * 4 * (bool(case.get("moved")) + bool(case.get("documents"))), "flops": 2 * flops}


# --------------------------------------------------------------------------- the same in 64 bits
def _family64(parents):
    """A token's line up to the root, by walking it."""
    up = parents.tolist()
    m = torch.zeros(len(up), len(up), dtype=torch.bool)
    for i in range(len(up)):
        j = i
        while j >= 0:
            m[i, j] = True
            j = up[j]
    return m


def _scores64(st, i, h, t0=0, t1=None):
    """One sequence's and one KV head's scores, [group][token][row] for tokens t0..t1."""
    n, b, tokens, d = st["lens"][i], st["begins"][i], st["tokens"], st["d"]
    t1 = tokens if t1 is None else t1
    heads = slice(h * st["group"], (h + 1) * st["group"])
    q = st["q"][i * tokens + t0:i * tokens + t1, heads].double()
    s = torch.einsum("tgd,rd->gtr", q, st["keys"][b:b + n, h].double()) / math.sqrt(d)
    cap = st["softcap"]
    if cap:
        s = torch.tanh(s / cap) * cap
    rp, qp = torch.arange(n, device=DEV), torch.arange(n - tokens + t0, n - tokens + t1, device=DEV)
    if "positions" in st:
        rp, qp = st["positions"][b:b + n].long(), st["q_positions"][i * tokens + t0:i * tokens + t1].long()
    hidden = None
    if st["op"] == "tree":
        m = _family64(st["parents"][i * tokens:(i + 1) * tokens]).to(DEV)
        depth = m.sum(1) - 1
        rp = torch.cat([rp[:n - tokens], n - tokens + depth])
        qp = n - tokens + depth
        hidden = torch.cat([torch.zeros(tokens, n - tokens, dtype=torch.bool, device=DEV), ~m], 1)
    diff = qp[:, None] - rp[None]
    no = diff < 0
    if st["window"]:
        no = no | (diff >= st["window"])
    if hidden is not None:
        no = no | hidden
    if "prefixes" in st:
        no = no & (rp >= st["prefixes"][i])[None]
    if "docs" in st:
        no = no | (st["docs"][b:b + n][None] != st["q_docs"][i * tokens + t0:i * tokens + t1][:, None])
    if "slopes" in st:
        s = s - st["slopes"][heads].double()[:, None, None] * diff.abs().double()
    s[:, no] = -math.inf
    return s


def exact(case, seed):
    if case["op"] == "evict":
        return _exact_evict(case, seed)
    st = prepare(case, seed) if case["op"] == "observe" else _inputs(case, seed)
    tokens, group = case["tokens"], case["group"]
    if case["op"] == "observe":
        w = st["weights_in"].double() * 0.5
        for i, (b, n) in enumerate(zip(st["begins"], st["lens"])):
            for h in range(case["kv_heads"]):
                lse = st["lse"][i * tokens:(i + 1) * tokens, h * group:(h + 1) * group].double().T
                p = torch.exp(_scores64(st, i, h) - lse[:, :, None])
                w[h, b:b + n] += torch.where(lse[:, :, None] > -math.inf, p, 0.0).sum((0, 1))
        return w
    out = torch.zeros(st["n_tokens"], st["n_heads"], case["d"], dtype=torch.float64, device=DEV)
    lse = torch.zeros(st["n_tokens"], st["n_heads"], dtype=torch.float64, device=DEV)
    for i, (b, n) in enumerate(zip(st["begins"], st["lens"])):
        for h in range(case["kv_heads"]):
            step = max(1, (1 << 27) // (n * group)) if case["op"] == "attend" else tokens
            for t0 in range(0, tokens, step):
                t1 = min(tokens, t0 + step)
                s = _scores64(st, i, h, t0, t1)
                z = torch.logsumexp(s, -1)
                p = torch.where(z[..., None] > -math.inf, torch.exp(s - z[..., None]), 0.0)
                at, hs = slice(i * tokens + t0, i * tokens + t1), slice(h * group, (h + 1) * group)
                out[at, hs] = torch.einsum("gtr,rd->tgd", p, st["values"][b:b + n, h].double())
                lse[at, hs] = z.T
    return out, lse


def _exact_evict(case, seed):
    """Row by row, as the rule says it (on the host)."""
    st = prepare(case, seed)
    to, budget = st["to"], case["budget"]
    for i, (b, n) in enumerate(zip(st["begins"], st["lens"])):
        for h in range(case["kv_heads"]):
            pos, w = st["positions"][h, b:b + n].tolist(), st["weights"][h, b:b + n].tolist()
            last = max(pos)
            rank = sorted(range(n), key=lambda r: (not (pos[r] < case["sink"] or last - pos[r] < case["recent"]), 0.0 if pos[r] < case["sink"] or last - pos[r] < case["recent"] else -w[r], r))
            keep = set(rank[:budget])
            late = iter(sorted(r for r in keep if r >= budget))
            src = torch.tensor([r if r in keep else next(late) for r in range(min(n, budget))], device=DEV)
            at = slice(i * budget, i * budget + len(src))
            to["keys"][at, h], to["values"][at, h] = st["keys"][b + src, h], st["values"][b + src, h]
            to["positions"][h, at], to["weights"][h, at] = st["positions"][h, b + src], st["weights"][h, b + src]
            if case["tiles"]:
                to["rows128"][h, at] = st["rows128"][h, b + src]
            to["source"][i, h, :len(src)] = src.to(torch.int32)
    return {**to, "keys": to["keys"].double(), "values": to["values"].double(), "weights": to["weights"].double()}
