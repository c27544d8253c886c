"""Cases and plain forms of the decoding operators (pero_ocr_amd.decode_ops): keys and values written to a paged cache in 8 bits
and read back, attention of drafted tokens over that cache, and the scores of given tokens.

With `own` false, run() computes an operator from elementary torch operations in 32 bits; with `own` true it makes the calls that
a decoding loop makes of pero_ocr_amd.decode_ops.  exact() computes the same in 64 bits, from the definitions.

The cache.  k, v: [pages, kv_heads, page_size, head_dim], either bfloat16 or float8_e4m3fn; slot s of a layer is row s % page_size
of page s // page_size.  An 8-bit row (one token, one head) has a scale of its own, the smallest power of two 2**(exp - 127) with
which its largest finite |value| becomes <= 448, exp >= 27; k_exp, v_exp: uint8 [pages, kv_heads, page_size]."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
GOLDEN = 0.6180339887498949


def listed():
    return [
        # one decoding step of 64 sequences: a row of every head each, launch-bound
        dict(name="write_step", op="write", tokens=64, kv_heads=8, head_dim=128, page=64, pages=640, dtype="bf16", cache="fp8", fused=True),
        # a long prompt filled in one call
        dict(name="write_fill", op="write", tokens=16384, kv_heads=8, head_dim=128, page=64, pages=320, dtype="bf16", cache="fp8", fused=False),
        # the encoder output of a batch of text lines (512 wide, 8 heads of 64), float32 rows sliced from the key / value projection
        dict(name="write_lines", op="write", tokens=5003, kv_heads=8, head_dim=64, page=16, pages=400, dtype="fp32", cache="fp8", fused=True),
        # a cached prefix read back for a second pass over it
        dict(name="read_prefix", op="read", tokens=16384, kv_heads=8, head_dim=128, page=64, pages=320, dtype="bf16", cache="fp8", holes=False),
        # rows of scattered lines in float32, some of them absent
        dict(name="read_lines", op="read", tokens=1009, kv_heads=8, head_dim=64, page=16, pages=128, dtype="fp32", cache="fp8", holes=True),
        # one step of 512 text lines over their cached positions, float32, as many key heads as query heads
        dict(name="attend_lines", op="attend", seqs=512, heads=8, kv_heads=8, head_dim=64, page=16, shortest=40, longest=272, fewest=1, most=1,
             tree=False, dtype="fp32", cache="fp8"),
        # one sequence verifies a tree of 33 drafted tokens
        dict(name="attend_tree", op="attend", seqs=1, heads=32, kv_heads=8, head_dim=128, page=64, shortest=4129, longest=4129, fewest=33, most=33,
             tree=True, dtype="bf16", cache="fp8"),
        # a batch of trees of several sizes over contexts of several lengths, cache in bfloat16
        dict(name="attend_trees", op="attend", seqs=24, heads=32, kv_heads=8, head_dim=128, page=64, shortest=517, longest=9001, fewest=7, most=64,
             tree=True, dtype="bf16", cache="bf16"),
        # single tokens over very long caches
        dict(name="attend_long", op="attend", seqs=4, heads=64, kv_heads=8, head_dim=128, page=128, shortest=60001, longest=131072, fewest=1, most=1,
             tree=False, dtype="bf16", cache="fp8"),
        # every frame of 256 text lines over the character set: the frame's symbol, its entropy, its rivals
        dict(name="score_frames", op="score", rows=36864, classes=232, top=4, dtype="fp32", banned=0.0),
        # a batch of sequences scored over a large vocabulary
        dict(name="score_vocab", op="score", rows=1024, classes=131072, top=20, dtype="bf16", banned=0.01),
        # the drafted tokens of one step over a large, odd vocabulary
        dict(name="score_step", op="score", rows=9, classes=151003, top=8, dtype="fp32", banned=0.01),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "score"])
    page = rng.choice([16, 32, 64, 128])
    if op in ("write", "read"):
        kv_heads, head_dim = rng.choice([1, 2, 3, 8, 16]), rng.choice([32, 64, 128, 256])
        tokens = _log_int(rng, 1, 16384 * 8 * 128 // (kv_heads * head_dim))
        case = dict(op=op, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, page=page, pages=-(-tokens // page) + rng.randint(1, 64),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), cache=rng.choice(["fp8", "fp8", "bf16"]))
        case["fused" if op == "write" else "holes"] = rng.random() < 0.5
        return case
    if op == "score":
        classes = _log_int(rng, 12, 152000)
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(60000, 1024 * 131072 // classes // 2))), classes=classes, top=rng.randint(0, min(24, classes)),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), banned=rng.choice([0.0, 0.01]))
    kv_heads, group, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8]), rng.choice([32, 64, 128, 256])
    tree = rng.random() < 0.6
    most = _log_int(rng, 1, 70)
    fewest = rng.randint(1, most)
    seqs = _log_int(rng, 1, 256)
    longest = min(131072, max(most, _log_int(rng, 1, max(2, 200_000_000 // (seqs * kv_heads * head_dim)))))
    # (the plain form holds every score of a batch at once; no more products than the largest listed case)
    longest = max(most, min(longest, 400_000_000 // (seqs * kv_heads * group * most), 16_000_000_000 // (seqs * kv_heads * group * most * head_dim)))
    return dict(op=op, seqs=seqs, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, page=page, shortest=rng.randint(most, longest), longest=longest,
                fewest=fewest, most=most, tree=tree, dtype=rng.choice(["bf16", "fp16", "fp32"]), cache=rng.choice(["fp8", "fp8", "bf16"]))


def _spread(lo, hi, n, shift=0.0):
    """n whole numbers spread over lo..hi, the largest first: a case's lengths are the same for every seed."""
    return [hi if i == 0 else lo + int((hi - lo + 1) * ((i * GOLDEN + shift) % 1.0)) for i in range(n)]


def _lengths(case):
    return _spread(case["shortest"], case["longest"], case["seqs"]), _spread(case["fewest"], case["most"], case["seqs"], 0.3)


def _quantise(x):
    """float32 [..., D] -> (e4m3 codes, uint8 exponents): the row's scale is the smallest power of two that brings it within 448."""
    fine = torch.isfinite(x)
    m, e = torch.frexp(torch.where(fine, x.abs(), 0.0).amax(-1))
    s = torch.where(m == 0, -100, e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-100)
    inverse = ((127 - s) << 23).to(torch.int32).view(torch.float32)
    codes = torch.where(fine, x * inverse[..., None], math.nan).to(torch.float8_e4m3fn)
    return codes, (s + 127).to(torch.uint8)


def _scale(exp):
    return (exp.to(torch.int32) << 23).view(torch.float32)


def _make_cache(case, pages, g):
    """A cache filled with keys and values whose rows differ in size, a few channels larger than the others."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    out = []
    for _ in range(2):
        rows = torch.randn(shape, device="cuda", generator=g)
        rows *= torch.exp2(torch.rand(shape[:3] + (1,), device="cuda", generator=g) * 3 - 2)
        rows *= torch.where(torch.arange(shape[3], device="cuda") % 37 == 5, 4.0, 1.0)
        out.append(_quantise(rows) if case["cache"] == "fp8" else (rows.to(torch.bfloat16), None))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _empty_cache(case):
    shape = (case["pages"], case["kv_heads"], case["page"], case["head_dim"])
    kind = DTYPES[case["cache"]]
    k, v = (torch.zeros(shape, dtype=torch.uint8 if case["cache"] == "fp8" else kind, device="cuda").view(kind) for _ in range(2))
    ke, ve = (torch.zeros(shape[:3], dtype=torch.uint8, device="cuda") if case["cache"] == "fp8" else None for _ in range(2))
    return k, v, ke, ve


def _tree_bits(counts, g):
    """Ancestor masks of random trees, int64 [tokens, words]: bit j of a row says that the token sees drafted token j of its sequence."""
    words = -(-max(counts) // 64)
    cpu = torch.Generator().manual_seed(int(torch.randint(0, 1 << 30, (1,), device="cuda", generator=g)))
    rows = []
    for n in counts:
        seen = []
        draws = torch.rand(n, generator=cpu).tolist()
        for i in range(n):
            parent = int(draws[i] * i) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        rows += [[(b >> 64 * w & (1 << 64) - 1) - (b >> 64 * w + 63 & 1) * (1 << 64) for w in range(words)] for b in seen]
    return torch.tensor(rows, dtype=torch.int64, device="cuda")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind = DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] in ("write", "read"):
        slots = torch.randperm(case["pages"] * case["page"], device="cuda", generator=g)[: case["tokens"]]
    if case["op"] == "write":
        heads, dim = case["kv_heads"], case["head_dim"]
        rows = torch.randn((case["tokens"], (3 if case["fused"] else 2) * heads, dim), device="cuda", generator=g)
        rows *= torch.where(torch.arange(dim, device="cuda") % 37 == 5, 4.0, 1.0)
        rows = rows.to(kind)
        k, v = (rows[:, -2 * heads:-heads], rows[:, -heads:]) if case["fused"] else (rows[:, :heads].contiguous(), rows[:, heads:].contiguous())
        return dict(state, k=k, v=v, slots=slots, cache=_empty_cache(case))
    if case["op"] == "read":
        if case["holes"]:
            slots[torch.rand(case["tokens"], device="cuda", generator=g) < 0.05] = -1
        return dict(state, slots=slots, cache=_make_cache(case, case["pages"], g))
    if case["op"] == "score":
        x = torch.randn((case["rows"], case["classes"]), device="cuda", generator=g)
        x *= torch.rand((case["rows"], 1), device="cuda", generator=g) * 3 + 1
        x = x.to(kind)
        tokens = torch.multinomial(torch.ones(case["classes"], device="cuda"), case["rows"], replacement=True, generator=g)
        if case["banned"]:
            x[:, torch.rand(case["classes"], device="cuda", generator=g) < case["banned"]] = -math.inf
        # the given symbol is the likeliest one in every other row
        best = x.float().amax(1, keepdim=True) if case["rows"] * case["classes"] < 1 << 24 else None
        if best is not None:
            tokens = torch.where(torch.arange(case["rows"], device="cuda") % 2 == 0, (x.float() == best).int().argmax(1), tokens)
        return dict(state, logits=x, tokens=tokens)
    lengths, counts = _lengths(case)
    need = [-(-n // case["page"]) for n in lengths]
    pages = sum(need) + 3
    ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(max(need), device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[at] = ids[: sum(need)]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    q = torch.randn((starts[-1], case["heads"], case["head_dim"]), device="cuda", generator=g).to(kind)
    return dict(state, q=q, cache=_make_cache(case, pages, g), table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), bits=_tree_bits(counts, g) if case["tree"] else None)


def _write(state):
    k, v, ke, ve = state["cache"]
    size = k.shape[2]
    page, row = state["slots"] // size, state["slots"] % size
    if ke is None:
        k[page, :, row] = state["k"].float().to(k.dtype)
        v[page, :, row] = state["v"].float().to(v.dtype)
    else:
        for data, exp, x in ((k, ke, state["k"]), (v, ve, state["v"])):
            codes, e = _quantise(x.float())
            data.view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
            exp[page, :, row] = e
    return state["cache"]


def _read(state):
    k, v, ke, ve = state["cache"]
    size, slots = k.shape[2], state["slots"]
    there = (slots >= 0)[:, None, None]
    page, row = slots.clamp(min=0) // size, slots.clamp(min=0) % size
    out = []
    for data, exp in ((k, ke), (v, ve)):
        x = data.view(torch.uint8)[page, :, row].view(data.dtype).float() * _scale(exp[page, :, row])[..., None] if exp is not None else data[page, :, row].float()
        out.append(torch.where(there, x, 0.0).to(DTYPES[state["case"]["dtype"]]))
    return tuple(out)


def _attend(state):
    case, q, (k, v, ke, ve), table = state["case"], state["q"], state["cache"], state["table"].clamp(min=0).long()
    seqs, most, hk = case["seqs"], case["most"], case["kv_heads"]
    total, heads, dim = q.shape
    group, span = heads // hk, table.shape[1] * case["page"]

    def rows(data, exp):
        x = data.view(torch.uint8)[table].view(data.dtype).float() * _scale(exp[table])[..., None] if exp is not None else data[table].float()
        return x.transpose(1, 2).reshape(seqs, hk, span, dim)

    starts, lengths = state["starts"].long(), state["lengths"].long()
    counts = starts[1:] - starts[:-1]
    lane = torch.arange(most, device=q.device)
    token = (starts[:-1, None] + lane).clamp(max=total - 1)
    padded = q.float()[token].view(seqs, most, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * most, dim)
    scores = (padded @ rows(k, ke).transpose(2, 3)).view(seqs, hk, group, most, span) * dim ** -0.5
    key = torch.arange(span, device=q.device)
    drafted = key[None, :] - (lengths - counts)[:, None]
    if state["bits"] is None:
        seen = drafted[:, None, :] <= lane[None, :, None]
    else:
        word = state["bits"][token].gather(2, (drafted.clamp(min=0, max=64 * state["bits"].shape[1] - 1) // 64)[:, None, :].expand(seqs, most, span))
        seen = (drafted[:, None, :] < 0) | (word >> (drafted.clamp(min=0) % 64)[:, None, :] & 1).bool()
    seen = (seen & (key[None, :] < lengths[:, None])[:, None, :])[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total_p = p.sum(-1, keepdim=True)
    p = p / torch.where(total_p == 0, 1.0, total_p)
    out = (p.view(seqs, hk, group * most, span) @ rows(v, ve)).view(seqs, heads, most, dim)
    lse = (top + torch.log(total_p)).view(seqs, heads, most)
    at = torch.arange(total, device=q.device)
    seq = (at[:, None] >= starts[None, 1:]).sum(1)
    return out[seq, :, at - starts[seq]].to(q.dtype), lse[seq, :, at - starts[seq]]


def _score(state):
    x, tokens, top = state["logits"].float(), state["tokens"], state["case"]["top"]
    best = x.amax(1, keepdim=True)
    e = torch.exp(x - best)
    z = e.sum(1, keepdim=True)
    entropy = torch.log(z) - torch.where(e > 0, e * (x - best), 0.0).sum(1, keepdim=True) / z
    lse = best + torch.log(z)
    # (a stable sort keeps equal logits in the order of their index)
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    return (x.gather(1, tokens[:, None]) - lse)[:, 0], entropy[:, 0], value[:, :top] - lse, index[:, :top].to(torch.int32)


def run(state):
    case = state["case"]
    if not own:
        return {"write": _write, "read": _read, "attend": _attend, "score": _score}[case["op"]](state)
    from pero_ocr_amd import decode_ops
    if case["op"] == "score":
        return decode_ops.token_logprobs(state["logits"], state["tokens"], top=case["top"])
    pages = decode_ops.KVPages(*state["cache"])
    if case["op"] == "write":
        decode_ops.kv_write(pages, state["k"], state["v"], state["slots"])
        return state["cache"]
    if case["op"] == "read":
        return decode_ops.kv_read(pages, state["slots"], dtype=DTYPES[case["dtype"]])
    return decode_ops.tree_attention(state["q"], pages, state["table"], state["lengths"], state["starts"], mask=state["bits"], max_queries=case["most"],
                                     want_lse=True)


def _bytes_of(name):
    return {"fp32": 4, "bf16": 2, "fp16": 2, "fp8": 1}[name]


def work(case):
    size = _bytes_of(case["dtype"])
    if case["op"] == "score":
        values = case["rows"] * case["classes"]
        return {"bytes": values * size + case["rows"] * (8 + 4 + 4 + 8 * case["top"]), "flops": 5 * values}
    row = case["head_dim"] * _bytes_of(case["cache"]) + (1 if case["cache"] == "fp8" else 0)
    if case["op"] in ("write", "read"):
        values = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": values * (row + case["head_dim"] * size) + 8 * case["tokens"], "flops": 2 * values * case["head_dim"]}
    lengths, counts = _lengths(case)
    keys = 2 * sum(lengths) * case["kv_heads"] * row
    queries = sum(counts) * case["heads"] * (2 * case["head_dim"] * size + 4)
    masks = 8 * sum(counts) * -(-case["most"] // 64) if case["tree"] else 0
    return {"bytes": keys + queries + masks + 4 * sum(-(-n // case["page"]) for n in lengths),
            "flops": 4 * case["head_dim"] * case["heads"] * sum(a * b for a, b in zip(lengths, counts))}


def _power64(n):
    """2.0 ** n in 64 bits for whole n, without a rounding (a power function may be off by the last bit)."""
    return (n.to(torch.int64) + 1023 << 52).view(torch.float64)


def _value64(codes, exp):
    x = codes.to(torch.float32).to(torch.float64)
    return x if exp is None else x * _power64(exp.to(torch.int64) - 127)[..., None]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "write":
        outs = []
        for x in (state["k"].double(), state["v"].double()):
            k = state["cache"][0]
            flat = torch.zeros((case["pages"] * case["page"], case["kv_heads"], case["head_dim"]), dtype=torch.float64, device="cuda")
            if case["cache"] == "fp8":
                biggest = x.abs().amax(2)
                power = torch.ceil(torch.log2((biggest / 448).clamp(min=2.0 ** -101)))
                # (the logarithm's own rounding may have moved a quotient next to a power of two across it)
                power = torch.where(biggest <= 448 * _power64(power - 1), power - 1, power)
                power = torch.where(biggest > 448 * _power64(power), power + 1, power)
                y = x / _power64(power.clamp(min=-100))[..., None]
                ulp = _power64(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
                flat[state["slots"]] = torch.round(y / ulp) * ulp
            else:
                ulp = _power64(torch.frexp(x.abs().clamp(min=2.0 ** -126))[1] - 8)
                flat[state["slots"]] = torch.round(x / ulp) * ulp
            outs.append(flat.view(k.shape[0], k.shape[2], k.shape[1], k.shape[3]).transpose(1, 2).contiguous())
        return outs[0], outs[1], None, None
    if case["op"] == "read":
        k, v, ke, ve = state["cache"]
        outs = []
        for data, exp in ((k, ke), (v, ve)):
            flat = _value64(data, exp).transpose(1, 2).reshape(-1, case["kv_heads"], case["head_dim"])
            out = flat[state["slots"].clamp(min=0)]
            out[state["slots"] < 0] = 0
            outs.append(out)
        return tuple(outs)
    if case["op"] == "score":
        outs = []
        for part in torch.split(torch.arange(case["rows"], device="cuda"), max(1, (1 << 27) // case["classes"])):
            x = state["logits"][part].double()
            logp = torch.log_softmax(x, dim=1)
            p = torch.exp(logp)
            given = logp[torch.arange(len(part), device="cuda"), state["tokens"][part]]
            best = torch.topk(logp, case["top"], dim=1).values
            outs.append((given, -torch.where(p > 0, p * logp, 0.0).sum(1), best))
        return torch.cat([o[0] for o in outs]), torch.cat([o[1] for o in outs]), torch.cat([o[2] for o in outs]), None
    k, v, ke, ve = state["cache"]
    lengths, counts = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    out, lse, first = [], [], 0
    for s, (length, n) in enumerate(zip(lengths, counts)):
        ids = state["table"][s, : -(-length // case["page"])].long()
        keys, values = (_value64(d[ids], None if e is None else e[ids]).transpose(0, 1).reshape(case["kv_heads"], -1, case["head_dim"])[:, :length]
                        for d, e in ((k, ke), (v, ve)))
        q = state["q"][first: first + n].double().transpose(0, 1).reshape(case["kv_heads"], group * n, case["head_dim"])
        scores = (torch.matmul(q, keys.transpose(1, 2).contiguous()) / math.sqrt(case["head_dim"])).view(case["kv_heads"], group, n, length)
        if state["bits"] is None:
            hidden = torch.ones((n, n), dtype=torch.bool, device="cuda").triu(1)
        else:
            j = torch.arange(n, device="cuda")
            hidden = (state["bits"][first: first + n][:, j // 64] >> j % 64 & 1) == 0
        scores[..., length - n:][..., hidden] = -math.inf
        sums = torch.logsumexp(scores, dim=3)
        out.append(torch.matmul(torch.exp(scores - sums[..., None]).view(case["kv_heads"], group * n, length), values)
                   .view(case["heads"], n, case["head_dim"]).transpose(0, 1))
        lse.append(sums.view(case["heads"], n).transpose(0, 1))
        first += n
    return torch.cat(out), torch.cat(lse)
