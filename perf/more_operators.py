"""Timed cases of a cache of key and value rows held in 4 bits and of what fills it: the norms and the position rotation of a layer's
query and key heads on their way into a cache, rows quantised as they are written and read back, and attention of decoded tokens, prompt
chunks and drafted trees over the 4-bit rows.

4 bits: blocks of 16 elements of a row of a head share a scale (float8 e4m3, of the block's largest size / 6); an element is one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (the even one of two in the low half of a byte), times the scale, times 2^exponent of the cache.
"""
import math

import torch

own = False

DEV = "cuda"
_stream = None  # the framework's calls are made on one stream of the caller's


def _rotate(**more):
    case = dict(op="rotate", dtype="bf16", d=128, kv_heads=8, group=4, seqs=1, tokens=1, rows=2048, rotary=128, interleaved=False, axes=1, norm=True, far=0)
    case.update(more)
    return case


def _attend(**more):
    case = dict(op="attend", dtype="bf16", d=128, kv_heads=8, group=4, seqs=1, rows=4096, ragged=False, tokens=1, softcap=0.0, alibi=False, window=0,
                prefix=0, documents=0, moved=False, tree=False, exponent=-3)
    case.update(more)
    return case


def listed():
    return [
        # One decoded token's heads on their way into the cache: what counts is the call itself.
        dict(_rotate(), name="rotate_decode"),
        # A prompt of text and images: positions of three axes.
        dict(_rotate(tokens=8192, rows=8192, axes=3), name="rotate_prompt_axes"),
        # float32 heads of a model that turns a part of each, far into several contexts, without norms.
        dict(_rotate(dtype="f32", d=96, kv_heads=4, group=3, seqs=5, tokens=37, rows=1501, rotary=64, interleaved=True, norm=False, far=1 << 20), name="rotate_f32_part"),
        # A batch of decoded tokens written to their caches, and what the caches then hold of them.
        dict(op="store", dtype="bf16", d=128, kv_heads=8, seqs=48, rows=2048, ragged=True, tokens=1, write=True, exponent=-3, name="store_decode"),
        # A long prompt written, and what attention will see of it.
        dict(op="store", dtype="bf16", d=128, kv_heads=8, seqs=1, rows=32768, ragged=False, tokens=32768, write=True, exponent=0, name="store_prompt"),
        # Rows of a batch of cached prompts back in float32, odd sizes.
        dict(op="store", dtype="f32", d=80, kv_heads=4, seqs=7, rows=9001, ragged=True, tokens=1, write=False, exponent=2, name="read_f32"),
        # One decoded token of a short conversation.
        dict(_attend(rows=512), name="decode_short"),
        # One decoded token on a long context, scores capped: the cache is read once.
        dict(_attend(rows=131072, softcap=50.0), name="decode_128k_softcap"),
        # A batch of decoded tokens with a distance bias; sequences of different lengths, rows kept by an earlier eviction.
        dict(_attend(seqs=48, rows=9001, ragged=True, alibi=True, moved=True), name="decode_batch_alibi"),
        # A chunk of a long prompt under a sliding window.
        dict(_attend(rows=16384, tokens=2048, window=4096, softcap=30.0), name="prompt_chunk_window"),
        # float32 queries: short continuations with a shared prefix that all of them see, odd sizes.
        dict(_attend(dtype="f32", d=96, kv_heads=4, group=3, seqs=5, rows=1501, ragged=True, tokens=37, prefix=129, alibi=True), name="chunk_f32_prefix"),
        # Drafted trees for a batch of sequences.
        dict(_attend(seqs=16, rows=8192, ragged=True, tokens=7, tree=True), name="tree_batch"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate"] * 3 + ["store"] * 3 + ["attend"] * 6)
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 4, 8])
    dtype, d = rng.choice(["bf16"] * 3 + ["f32"]), rng.choice([64, 80, 96, 128, 128, 128, 256])
    seqs, ragged = _spread(rng, 1, 64), rng.random() < 0.6
    most = (1 << 20) // d * 128 // kv_heads // seqs  # rows of a sequence
    if op == "rotate":
        tokens = max(1, min(_spread(rng, 1, 8192), 8192 * 4096 // (seqs * kv_heads * (group + 1) * d)))
        rotary = rng.choice([d, d, d // 2])
        return _rotate(dtype=dtype, d=d, kv_heads=kv_heads, group=group, seqs=seqs, tokens=tokens, rows=max(tokens, min(most, _spread(rng, 16, 4096))), rotary=rotary,
                       interleaved=rng.random() < 0.3, axes=rng.choice([1, 1, 3, 4]), norm=rng.random() < 0.7, far=rng.choice([0, 0, 1]) * _spread(rng, 1, 1 << 22))
    exponent = rng.choice([-4, -3, -1, 0, 0, 2])
    if op == "store":
        rows = max(1, min(most * 2 // 5, _spread(rng, 1, 65536)))
        return dict(op=op, dtype=dtype, d=d, kv_heads=kv_heads, seqs=seqs, rows=rows, ragged=ragged, tokens=max(1, min(rows // 3, _spread(rng, 1, rows + 1))), write=rng.random() < 0.6,
                    exponent=exponent)
    case = dict(dtype=dtype, d=d, kv_heads=kv_heads, group=group, ragged=ragged, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                window=rng.choice([0, 0, 0, 1]) * _spread(rng, 16, 4096), exponent=exponent)
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "tree"])
    if kind == "tree":
        tokens = _spread(rng, 1, 64)
        seqs = min(seqs, 16)
        rows = max(tokens, min(most, (1 << 22) // (seqs * tokens), _spread(rng, 64, 65536)))
        return _attend(seqs=seqs, rows=rows, tokens=tokens, tree=True, **case)
    tokens = _spread(rng, 5, 4096) if kind == "chunk" else rng.choice([1, 1, 1, 2, 3])
    if kind == "chunk":
        seqs = min(seqs, 8)
        pairs = (1 << 25) if dtype == "f32" else (1 << 27)  # (head, token, row) triples stay below the largest listed case's
        tokens = max(1, min(tokens, int(math.sqrt(pairs / (seqs * kv_heads * group)))))
        rows = min(most, max(tokens, _spread(rng, tokens, max(tokens + 1, pairs // (seqs * kv_heads * group * tokens)))))
    else:
        rows = min(most, _spread(rng, tokens + 1, 131072))
    return _attend(seqs=seqs, rows=max(rows, tokens), tokens=tokens, alibi=rng.random() < 0.3, prefix=rng.choice([0, 0, 1]) * _spread(rng, 1, max(rows, 1)),
                   documents=rng.choice([0, 0, 2, 7]), moved=rng.random() < 0.3, **case)


# --------------------------------------------------------------------------- inputs
def _lengths(case):
    n, low = case["rows"], max(case["tokens"], case["rows"] // 3)
    return [n - ((i * 40503 + 17) % 65536) * (n - low) // 65536 if case.get("ragged") else n for i in range(case["seqs"])]


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


def _scale_bytes(d):
    return 4 if d <= 64 else 8 if d <= 128 else 16


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
    at = parents.long()
    link = torch.zeros(seqs, tokens, tokens, device=DEV)
    link.scatter_(2, at.clamp(min=0)[:, :, None], (at >= 0).float()[:, :, None])
    reach = torch.eye(tokens, device=DEV).repeat(seqs, 1, 1)
    for _ in range(max(1, math.ceil(math.log2(tokens + 1)))):  # each time twice as far up the tree
        reach = ((reach + link @ reach) > 0).float()
        link = ((link @ link) > 0).float()
    return reach > 0


def _axis_of_pair(case):
    """The axis by which each of a head's turned pairs goes: in runs (the first axis' is half as long) or, interleaved, in turn."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    at = torch.arange(pairs, device=DEV)
    if case["interleaved"]:
        return (at % axes).to(torch.uint8)
    return ((at * (2 * axes - 1) // pairs + 1) // 2).clamp(max=axes - 1).to(torch.uint8)


def _rotate_inputs(case, seed):
    gen, lens, dtype, d = _gen(seed), _lengths(case), _type(case), case["d"]
    begins = _begins(lens)
    n, tokens, kv, heads = case["seqs"] * case["tokens"], case["tokens"], case["kv_heads"], case["kv_heads"] * case["group"]
    st = dict(case, lens=lens, begins=begins, total=begins[-1], n_tokens=n, n_heads=heads)
    st["qkv"] = (torch.randn(n, (heads + 2 * kv) * d, generator=gen, device=DEV) * torch.exp(0.5 * torch.randn((heads + 2 * kv) * d, generator=gen, device=DEV))).to(dtype)
    parts = st["qkv"].view(n, heads + 2 * kv, d).split([heads, kv, kv], 1)
    st["q"], st["k"], st["v"] = parts
    st["q_weight"], st["k_weight"] = (1 + 0.3 * torch.randn(d, generator=gen, device=DEV) for _ in range(2))
    st["freq"] = (10000.0 ** (-torch.arange(case["rotary"] // 2, device=DEV, dtype=torch.float64) / (case["rotary"] // 2))).float()
    st["axis"] = _axis_of_pair(case)
    first = torch.tensor(lens, device=DEV)[:, None] - tokens + case["far"] + torch.arange(tokens, device=DEV)
    pos = first.reshape(-1).repeat(case["axes"], 1)
    if case["axes"] > 1:  # rows and columns of images beside the running number
        pos[1:] = torch.randint(0, 64, (case["axes"] - 1, n), generator=gen, device=DEV) + pos[:1] // 2
    st["positions"] = pos.to(torch.int32).contiguous()
    st["rows_of"] = (torch.tensor(begins[1:], device=DEV)[:, None] - tokens + torch.arange(tokens, device=DEV)).reshape(-1)
    st["q_out"] = torch.empty(n, heads, d, dtype=dtype, device=DEV)
    st["keys"], st["values"] = (torch.zeros(st["total"], kv, d, dtype=dtype, device=DEV) for _ in range(2))
    return st


def _pack(x, exponent):
    """Codes and scales, as bytes, of rows x [row][head][d]: both laid out [head][row]."""
    code, scale = _quantised(x, exponent)
    rows, heads, d = x.shape
    byte = (code.view(rows, heads, d // 2, 2) * torch.tensor([1, 16], device=DEV)).sum(3).to(torch.uint8)
    room = torch.zeros(heads, rows, _scale_bytes(d), dtype=torch.uint8, device=DEV)
    room[:, :, :d // 16] = scale.permute(1, 0, 2)
    wide = torch.zeros(heads, rows, -(-d // 32) * 16, dtype=torch.uint8, device=DEV)
    wide[:, :, :d // 2] = byte.permute(1, 0, 2)
    return wide, room


def _inputs(case, seed):
    if case["op"] == "rotate":
        return _rotate_inputs(case, seed)
    gen, lens, tokens, dtype = _gen(seed), _lengths(case), case["tokens"], _type(case)
    begins = _begins(lens)
    total, heads, d = begins[-1], case["kv_heads"], case["d"]
    chan = torch.exp(0.5 * torch.randn(d, generator=gen, device=DEV))
    st = dict(case, lens=lens, begins=begins, total=total)
    fresh = case["op"] == "store" and case["write"]  # what is written, else what the cache holds
    n = case["seqs"] * tokens if fresh else total
    keys = (torch.randn(n, heads, d, generator=gen, device=DEV) * chan).to(dtype)
    values = torch.randn(n, heads, d, generator=gen, device=DEV).mul_(0.5).to(dtype)
    if fresh:
        st["k"], st["v"] = keys, values
        st["codes"] = [torch.zeros(heads, total, -(-d // 32) * 16, dtype=torch.uint8, device=DEV) for _ in range(2)]
        st["scales"] = [torch.zeros(heads, total, _scale_bytes(d), dtype=torch.uint8, device=DEV) for _ in range(2)]
    else:
        (kc, ks), (vc, vs) = _pack(keys, case["exponent"]), _pack(values, case["exponent"])
        st["codes"], st["scales"] = [kc, vc], [ks, vs]
    if case["op"] == "store":
        st["keys"], st["values"] = (torch.empty(n, heads, d, dtype=dtype, device=DEV) for _ in range(2))
        return st
    n_heads = heads * case["group"]
    st["n_heads"], st["n_tokens"] = n_heads, case["seqs"] * tokens
    st["q"] = (torch.randn(case["seqs"] * tokens, n_heads, d, generator=gen, device=DEV) * 1.5).to(dtype)
    if case["moved"]:
        # rows that an eviction has left, in another order than they were written
        gaps = [torch.cumsum(torch.randint(1, 4, (n,), generator=gen, device=DEV), 0) for n in lens]
        mixed = [torch.cat([g[torch.randperm(n - tokens, generator=gen, device=DEV)], g[n - tokens:]]) for g, n in zip(gaps, lens)]
        st["positions"] = torch.cat(mixed).to(torch.int32)
        st["q_positions"] = torch.cat([g[-tokens:] for g in mixed]).to(torch.int32)
    if case["documents"]:
        st["docs"] = torch.cat([_documents(gen, n, case["documents"]) for n in lens])
        st["q_docs"] = torch.cat([st["docs"][b - tokens:b] for b in begins[1:]])
    if case["alibi"]:
        st["slopes"] = (2.0 ** (-8.0 * torch.arange(1, n_heads + 1, device=DEV) / n_heads)).float()
    if case["prefix"]:
        st["prefixes"] = torch.tensor([min(case["prefix"], n) for n in lens], dtype=torch.int32, device=DEV)
    if case["tree"]:
        st["parents"] = torch.cat([_parents(gen, tokens) for _ in lens])
    st["out"] = torch.empty(st["n_tokens"], n_heads, d, dtype=dtype, device=DEV)
    st["lse"] = torch.empty(st["n_tokens"], n_heads, device=DEV)
    return st


def prepare(case, seed):
    global _stream
    st = _inputs(case, seed)
    if own:  # the handles that a program keeps: where its cache lies, where its tokens come to lie, the table of its sequences
        import slhav2_b200 as S

        if _stream is None:
            _stream = torch.cuda.Stream()
        S.set_stream(_stream.cuda_stream)
        torch.cuda.synchronize()
        dtype, tokens, d, kv = S.BF16 if case["dtype"] == "bf16" else S.F32, case["tokens"], case["d"], case["kv_heads"]
        st["segs"] = S.make_segments([(b, n, i * tokens, tokens, 0) for i, (b, n) in enumerate(zip(st["begins"], st["lens"]))])
        if case["op"] == "rotate":
            wide = st["qkv"].stride(0)
            st["heads"] = S.HeadRows(st["q"], st["k"], st["v"], st["n_tokens"], st["n_heads"], kv, d, dtype=dtype, token_stride=wide, head_stride=d, norm=case["norm"], eps=1e-6,
                                     q_weight=st["q_weight"] if case["norm"] else None, k_weight=st["k_weight"] if case["norm"] else None)
            st["turn"] = S.Rotation(st["freq"], st["positions"], case["rotary"], n_axes=case["axes"], axes=st["axis"] if case["axes"] > 1 else None, interleaved=case["interleaved"])
            st["cache"] = S.KvCache(st["keys"], st["values"], kv, d, dtype=dtype)
            return st
        (kc, vc), (ks, vs), total = st["codes"], st["scales"], st["total"]
        st["cache4"] = S.KvCache4(kc, vc, ks, vs, kv, d, dtype=dtype, code_row_stride=kc.shape[2], code_head_stride=total * kc.shape[2], scale_row_stride=ks.shape[2],
                                  scale_head_stride=total * ks.shape[2], key_exponent=case["exponent"], value_exponent=case["exponent"], positions=st.get("positions"),
                                  documents=st.get("docs"))
        if case["op"] == "store":
            st["to"] = S.KvCache(st["keys"], st["values"], kv, d, dtype=dtype)
            if case["write"]:
                st["from"] = S.KvCache(st["k"], st["v"], kv, d, dtype=dtype)
                st["read_segs"] = S.make_segments([(e - tokens, tokens, 0, 0, 0) for e in st["begins"][1:]])
                st["to_segs"] = S.make_segments([(i * tokens, tokens, 0, 0, 0) for i in range(case["seqs"])])
            return st
        st["queries"] = S.CacheQueries(st["q"], st["n_tokens"], st["n_heads"], d, softcap=case["softcap"], window=case["window"], slopes=st.get("slopes"),
                                       prefix=st.get("prefixes"), positions=st.get("q_positions"), documents=st.get("q_docs"))
    return st


# --------------------------------------------------------------------------- plain forms
def _plain_rotate(st):
    d, r = st["d"], st["rotary"]
    turns = st["positions"][st["axis"].long()].double().T * st["freq"].double()  # [token][pair], in 64 bits: far positions' angles
    cos, sin = torch.cos(turns).float()[:, None], torch.sin(turns).float()[:, None]

    def turned(x, weight):
        x = x.float()
        if st["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if st["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        one, two = a * cos - b * sin, a * sin + b * cos
        both = torch.stack([one, two], -1).flatten(-2) if st["interleaved"] else torch.cat([one, two], -1)
        return torch.cat([both, x[..., r:]], -1) if r < d else both

    st["q_out"].copy_(turned(st["q"], st["q_weight"]))
    st["keys"][st["rows_of"]] = turned(st["k"], st["k_weight"]).to(st["keys"].dtype)
    st["values"][st["rows_of"]] = st["v"]
    return st["q_out"], st["keys"], st["values"]


def _nearest(x, least, bits):
    """x >= 0 rounded to `bits` binary places behind the first one, ties to even; below 2^least in steps as there."""
    e = torch.frexp(x).exponent.clamp(min=least + 1) - 1
    step = torch.ldexp(torch.ones_like(x), e - bits)
    return torch.round(x / step) * step


def _quantised(x, exponent):
    """[row][head][d] -> each element's four bits and each block's scale as a byte; in 64 bits, as an element may lie next to a border."""
    blocks = x.double().unflatten(-1, (-1, 16)) * 2.0 ** -exponent
    size = blocks.abs()
    scale = _nearest(size.amax(-1) / 6, -6, 3).clamp(max=448.0)
    held = _nearest(size / torch.where(scale > 0, scale, 1.0)[..., None], 0, 1).clamp(max=6.0) * (scale > 0)[..., None]
    code = torch.where(held < 2, held * 2, torch.where(held < 4, held + 2, held / 2 + 4))
    code = code.long() + 8 * (blocks < 0)
    e = torch.frexp(scale).exponent.clamp(min=-5) - 1  # e4m3: four bits of exponent (bias 7), three of fraction
    byte = torch.where(scale < 2.0 ** -6, scale * 512, (e + 6) * 8 + scale * torch.ldexp(torch.full_like(scale, 8.0), -e))
    return code.flatten(-2), byte.long()


def _values_of(codes, scales, d, exponent):
    """[head][row] bytes -> the values that they stand for, [row][head][d] float32."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV)
    table = torch.cat([table, -table])
    code = codes[:, :, :d // 2]
    held = torch.stack([table[(code & 15).long()], table[(code >> 4).long()]], -1).flatten(-2)
    byte = scales[:, :, :d // 16].float()
    e = torch.floor(byte / 8)
    scale = torch.where(e > 0, torch.exp2(e - 7) * (1 + (byte - 8 * e) / 8), byte / 512)
    return (held.unflatten(-1, (-1, 16)) * (scale * 2.0 ** exponent)[..., None]).flatten(-2).permute(1, 0, 2)


def _plain_store(st):
    d, e = st["d"], st["exponent"]
    if st["write"]:
        tokens = st["tokens"]
        rows = (torch.tensor(st["begins"][1:], device=DEV)[:, None] - tokens + torch.arange(tokens, device=DEV)).reshape(-1)
        (kc, ks), (vc, vs) = _pack(st["k"], e), _pack(st["v"], e)
        st["codes"][0][:, rows], st["codes"][1][:, rows] = kc, vc
        st["scales"][0][:, rows], st["scales"][1][:, rows] = ks, vs
        codes, scales = [c[:, rows] for c in st["codes"]], [s[:, rows] for s in st["scales"]]
    else:
        codes, scales = st["codes"], st["scales"]
    st["keys"].copy_(_values_of(codes[0], scales[0], d, e))
    st["values"].copy_(_values_of(codes[1], scales[1], d, e))
    return st["keys"], st["values"]


def _seen(st, at, there):
    """[sequence][token][row]: the rows that a token sees, and the distance between the two."""
    seqs, tokens = st["seqs"], st["tokens"]
    lens = torch.tensor(st["lens"], device=DEV)
    where = torch.where(there, torch.tensor(st["begins"][:-1], device=DEV)[:, None] + at, 0)
    if st["moved"]:
        row_pos, q_pos = st["positions"][where].long(), st["q_positions"].long().view(seqs, tokens)
    else:
        row_pos, q_pos = at.expand(seqs, -1), lens[:, None] - tokens + torch.arange(tokens, device=DEV)
    drafted = None
    if st["tree"]:
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
    return where, seen & there[:, None, :], away


def _plain_attend(st):
    seqs, tokens, heads, d = st["seqs"], st["tokens"], st["kv_heads"], st["d"]
    lens = torch.tensor(st["lens"], device=DEV)
    at = torch.arange(max(st["lens"]), device=DEV)
    where, seen, away = _seen(st, at, at < lens[:, None])
    q = st["q"].float().view(seqs, tokens, heads, -1, d).permute(0, 2, 3, 1, 4)
    group, n = q.shape[2], where.shape[1]
    k = _values_of(st["codes"][0], st["scales"][0], d, st["exponent"])[where].permute(0, 2, 3, 1)  # [sequence][kv_head][d][row]
    s = torch.matmul(q.reshape(seqs, heads, group * tokens, d), k).view(seqs, heads, group, tokens, n) * d ** -0.5
    del k
    if st["softcap"]:
        s = st["softcap"] * torch.tanh(s / st["softcap"])
    if "slopes" in st:
        s -= st["slopes"].view(1, heads, group, 1, 1) * away.abs().float()[:, None, None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1)
    lse = torch.log(total) + top[..., 0]
    v = _values_of(st["codes"][1], st["scales"][1], d, st["exponent"])[where].permute(0, 2, 1, 3)  # [sequence][kv_head][row][d]
    o = torch.matmul(p.view(seqs, heads, group * tokens, n), v).view(seqs, heads, group, tokens, d)
    o /= torch.where(total > 0, total, 1.0)[..., None]
    st["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(st["out"].shape))
    st["lse"].copy_(lse.permute(0, 3, 1, 2).reshape(st["lse"].shape))
    return st["out"], st["lse"]


def run(st):
    op = st["op"]
    if own:
        import slhav2_b200 as S

        if op == "rotate":
            S.rotate_heads(st["heads"], st["turn"], q_out=st["q_out"], to=st["cache"], segments=st["segs"])
            return st["q_out"], st["keys"], st["values"]
        if op == "store":
            if st["write"]:
                S.write_cache4(st["cache4"], st["segs"], st["from"], len(st["k"]))
                S.read_cache4(st["cache4"], st["read_segs"], st["to"], st["to_segs"])
            else:
                S.read_cache4(st["cache4"], st["segs"], st["to"])
            return st["keys"], st["values"]
        if st["tree"]:
            S.attend_tree4(st["cache4"], st["segs"], st["queries"], st["parents"], st["out"], st["lse"])
        else:
            S.attend_cache4(st["cache4"], st["segs"], st["queries"], st["out"], st["lse"])
        return st["out"], st["lse"]
    return _plain_rotate(st) if op == "rotate" else _plain_store(st) if op == "store" else _plain_attend(st)


# --------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """(token, row) pairs that are seen, about, and the rows that any token sees."""
    pairs, rows = 0.0, 0
    tokens, window, prefix = case["tokens"], case["window"], case["prefix"]
    for n in _lengths(case):
        ctx = n - tokens
        span = min(window, n) if window and not case["moved"] else n
        seen = sum(min(ctx + t + 1, span) for t in range(tokens)) if tokens <= 4096 else tokens * (ctx + (tokens + 1) / 2)
        docs = max(1, case["documents"])
        if docs > 1:
            # a token sees its document's earlier rows: of runs cut at random, twice the share of equal ones
            seen = min(seen, tokens * 2.0 * n / (docs + 1) / 2)
        seen = max(seen, float(min(prefix, n)) * tokens / docs)
        pairs += min(seen, float(tokens) * n)
        rows += n if docs > 1 or not window else min(n, span + tokens - 1 + min(prefix, n))
    return pairs, rows


def work(case):
    e, d, heads = (2 if case["dtype"] == "bf16" else 4), case["d"], case["kv_heads"]
    n = case["seqs"] * case["tokens"]
    if case["op"] == "rotate":
        # every head in and out once; a norm's square, factor and weight and a turn's two products and sum for each element of queries and keys
        turned = n * heads * (case["group"] + 1) * d
        return {"bytes": 2 * e * n * heads * (case["group"] + 2) * d + 4 * n * case["axes"], "flops": turned * (3 + 4 * case["norm"])}
    held = d // 2 + d // 16
    if case["op"] == "store":
        rows = n if case["write"] else sum(_lengths(case))
        return {"bytes": 2 * rows * heads * (held + d * e + (d * e if case["write"] else 0)), "flops": 2 * rows * heads * d * (3 if case["write"] else 1)}
    pairs, rows = _pairs(case)
    n_q = n * heads * case["group"]
    return {"bytes": 2 * heads * rows * held + n_q * (2 * d * e + 4) + rows * 4 * (case["moved"] + bool(case["documents"])),
            "flops": 4 * pairs * heads * case["group"] * d}


# --------------------------------------------------------------------------- the same in 64 bits
def _exact_rotate(case, seed):
    st = _inputs(case, seed)
    r, n = case["rotary"], st["n_tokens"]
    q, k, v = (x.double().clone() for x in (st["q"], st["k"], st["v"]))
    if case["norm"]:
        for x, w in ((q, st["q_weight"]), (k, st["k_weight"])):
            x /= torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["d"] + 1e-6)
            x *= w.double()
    for p in range(r // 2):  # pair by pair
        angle = st["positions"][int(st["axis"][p])].double() * float(st["freq"][p])
        c, s = torch.cos(angle).view(n, 1), torch.sin(angle).view(n, 1)
        i, j = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + r // 2)
        for x in (q, k):
            a, b = x[:, :, i].clone(), x[:, :, j].clone()
            x[:, :, i], x[:, :, j] = c * a - s * b, s * a + c * b
    keys, values = st["keys"].double(), st["values"].double()
    keys[st["rows_of"]], values[st["rows_of"]] = k, v
    return q, keys, values


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_E4M3 = [m / 512 if e == 0 else 2.0 ** (e - 7) * (1 + m / 8) for e in range(16) for m in range(8)][:127]


def _to_list(x, values):
    """The place of the nearest of `values` (rising) for each x >= 0; a tie goes to the even place."""
    v = torch.tensor(values, dtype=torch.float64, device=DEV)
    mid = (v[1:] + v[:-1]) / 2
    low, high = torch.bucketize(x, mid), torch.bucketize(x, mid, right=True)
    return torch.where(low % 2 == 0, low, high)


def _round_trip64(x, exponent):
    """What rows read back as, from the list of values and the distances to them."""
    y = x.double() / 2.0 ** exponent
    y = y.reshape(*y.shape[:-1], -1, 16)
    s = torch.tensor(_E4M3, dtype=torch.float64, device=DEV)[_to_list(y.abs().max(-1).values / 6, _E4M3)][..., None]
    held = torch.tensor(_E2M1, dtype=torch.float64, device=DEV)[_to_list(y.abs() / s, _E2M1)]
    return (torch.where(s > 0, torch.sign(y) * held * s, 0.0) * 2.0 ** exponent).reshape(x.shape)


def _table64(codes, scales, d, exponent):
    """Rows [row][d] of one head's bytes, by tables over whole bytes."""
    pair = torch.tensor([[(-1.0 if c & 8 else 1.0) * _E2M1[c & 7] for c in (b & 15, b >> 4)] for b in range(256)], dtype=torch.float64, device=DEV)
    s = torch.tensor(_E4M3, dtype=torch.float64, device=DEV)[scales[:, :d // 16].long()]
    held = pair[codes[:, :d // 2].long()].reshape(len(codes), d)
    return held * s.repeat_interleave(16, 1) * 2.0 ** exponent


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


def _scores64(st, k, i, h, t0, t1):
    """One sequence's and one KV head's scores, [group][token][row] for tokens t0..t1; k: its rows."""
    n, b, tokens, d = st["lens"][i], st["begins"][i], st["tokens"], st["d"]
    heads = slice(h * st["group"], (h + 1) * st["group"])
    q = st["q"][i * tokens + t0:i * tokens + t1, heads].double()
    s = torch.einsum("tgd,rd->gtr", q, k) / math.sqrt(d)
    cap = st["softcap"]
    if cap:
        s = torch.tanh(s / cap) * cap
    rp, qp = torch.arange(n, device=DEV), torch.arange(n - tokens + t0, n - tokens + t1, device=DEV)
    if st["moved"]:
        rp, qp = st["positions"][b:b + n].long(), st["q_positions"][i * tokens + t0:i * tokens + t1].long()
    hidden = None
    if st["tree"]:
        m = _family64(st["parents"][i * tokens:(i + 1) * tokens]).to(DEV)
        depth = m.sum(1) - 1
        rp = torch.cat([rp[:n - tokens], n - tokens + depth])
        qp = n - tokens + depth[t0:t1]
        hidden = torch.cat([torch.zeros(t1 - t0, n - tokens, dtype=torch.bool, device=DEV), ~m[t0:t1]], 1)
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
    if case["op"] == "rotate":
        return _exact_rotate(case, seed)
    st = _inputs(case, seed)
    d, e = case["d"], case["exponent"]
    if case["op"] == "store":
        if case["write"]:
            return _round_trip64(st["k"], e), _round_trip64(st["v"], e)
        return tuple(torch.stack([_table64(st["codes"][x][h], st["scales"][x][h], d, e) for h in range(case["kv_heads"])], 1) for x in range(2))
    tokens, group = case["tokens"], case["group"]
    out = torch.zeros(st["n_tokens"], st["n_heads"], d, dtype=torch.float64, device=DEV)
    lse = torch.zeros(st["n_tokens"], st["n_heads"], dtype=torch.float64, device=DEV)
    for h in range(case["kv_heads"]):
        keys, values = (_table64(st["codes"][x][h], st["scales"][x][h], d, e) for x in range(2))
        for i, (b, n) in enumerate(zip(st["begins"], st["lens"])):
            step = max(1, (1 << 27) // (n * group))
            for t0 in range(0, tokens, step):
                t1 = min(tokens, t0 + step)
                s = _scores64(st, keys[b:b + n], i, h, t0, t1)
                z = torch.logsumexp(s, -1)
                p = torch.where(z[..., None] > -math.inf, torch.exp(s - z[..., None]), 0.0)
                at, hs = slice(i * tokens + t0, i * tokens + t1), slice(h * group, (h + 1) * group)
                out[at, hs] = torch.einsum("gtr,rd->tgd", p, values[b:b + n])
                lse[at, hs] = z.T
    return out, lse
