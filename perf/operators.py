"""The attention operators of a serving loop, as workloads: cases, inputs, the
plain form of each, and the calls a user's program makes of them.

* ``slots``: block tables and slot maps from request lengths (``assign_slots``).
* ``write``: K/V rows into a paged cache at those slots (``write_cache``).
* ``prompt``: attention over packed prompts (``varlen_attention``).
* ``tree``: attention of drafted tokens over the paged cache
  (``tree_attention``); one token per request is plain decoding.

The lengths of a batch and the shape of a draft tree follow from the case
alone, so its work is known without its inputs; block ids and values come from
the seed.  Caches hold more blocks than the batch uses, in shuffled order.
"""

import random

import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}


def _slots(name, B, lo, hi, new_lo, new_hi, block, pad=0):
    return {"name": name, "op": "slots", "B": B, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi,
            "block": block, "pad": pad}


def _write(name, dtype, T, HK, D, block, layout="bshd", pad=0):
    return {"name": name, "op": "write", "dtype": dtype, "T": T, "HK": HK, "D": D, "block": block, "layout": layout,
            "pad": pad}


def _prompt(name, dtype, B, lo, hi, HQ, HK, D, prefix=0, causal=True, packed=False):
    return {"name": name, "op": "prompt", "dtype": dtype, "B": B, "lo": lo, "hi": hi, "HQ": HQ, "HK": HK, "D": D,
            "prefix": prefix, "causal": causal, "packed": packed}


def _tree(name, dtype, B, lo, hi, nodes, tree, HQ, HK, D, block, layout="bshd"):
    return {"name": name, "op": "tree", "dtype": dtype, "B": B, "lo": lo, "hi": hi, "nodes": nodes, "tree": tree,
            "HQ": HQ, "HK": HK, "D": D, "block": block, "layout": layout}


def listed():
    return [
        # The bookkeeping of one decoding step of 64 requests.
        _slots("slots_decode_b64", 64, 1, 8192, 1, 1, 16),
        # A large batch of prompts entering the cache, padded to a captured graph's size.
        _slots("slots_prompts_b512", 512, 0, 100, 1, 1024, 64, pad=1000),
        # One decoding step's K and V rows, one layer.
        _write("write_bf16_t64", "bf16", 64, 8, 128, 16),
        # A batch of prompts' K and V rows, one layer, into blocks held head by head.
        _write("write_bf16_t16384", "bf16", 16384, 8, 128, 16, layout="bhsd", pad=37),
        # A single short prompt: latency.
        _prompt("prompt_bf16_1x197", "bf16", 1, 197, 197, 16, 4, 128),
        # A batch of uneven prompts, read in place from one fused q/k/v projection.
        _prompt("prompt_bf16_8x200_4096", "bf16", 8, 200, 4096, 32, 8, 128, packed=True),
        # Chunks of prompts behind cached prefixes, head dim 64.
        _prompt("prompt_f16_d64_16x64_1100", "f16", 16, 64, 1100, 16, 4, 64, prefix=1000),
        # One long prompt with many heads: the largest product.
        _prompt("prompt_bf16_1x16384", "bf16", 1, 16384, 16384, 64, 8, 128),
        # One user, a short conversation, one token at a time: latency.
        _tree("decode_bf16_b1_s700", "bf16", 1, 700, 700, 1, False, 64, 8, 128, 16),
        # A serving batch, one token per request, uneven contexts.
        _tree("decode_bf16_b64_s8192", "bf16", 64, 100, 8192, 1, False, 64, 8, 128, 16),
        # Verification of drafted trees of up to 48 nodes for 16 requests.
        _tree("tree_bf16_b16_n48", "bf16", 16, 500, 12000, 48, True, 32, 8, 128, 32),
        # A chain of 5 drafted tokens over one long document, head dim 64.
        _tree("chain_f16_d64_s131072", "f16", 1, 131072, 131072, 5, False, 32, 4, 64, 64, layout="bhsd"),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["slots", "write", "prompt", "prompt", "prompt", "tree", "tree", "tree"])
    while True:
        hk, group, d = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 128])
        dtype, block = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
        layout = rng.choice(["bshd", "bhsd"])
        if op == "slots":
            lo, new = _log(rng, 1, 4096) - 1, _log(rng, 1, 2048)
            case = _slots("", _log(rng, 1, 1024), lo, lo + _log(rng, 1, 8192), rng.choice([0, 1, new]), new, block,
                          pad=rng.choice([0, 0, _log(rng, 1, 1000)]))
        elif op == "write":
            case = _write("", dtype, _log(rng, 1, 16384), hk, d, block, layout, pad=rng.choice([0, 0, _log(rng, 1, 100)]))
        elif op == "prompt":
            lo = _log(rng, 1, 8192)
            hi = rng.choice([lo, _log(rng, lo, 16384)])
            case = _prompt("", dtype, _log(rng, 1, 64), lo, hi, hk * group, hk, d,
                           prefix=rng.choice([0, 0, _log(rng, 1, 4096)]), causal=rng.random() < 0.8,
                           packed=rng.random() < 0.5)
        else:
            lo = _log(rng, 1, 32768) - 1
            hi = rng.choice([lo, _log(rng, lo + 1, 131072)])
            nodes = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 130)])
            case = _tree("", dtype, _log(rng, 1, 128), lo, hi, nodes, nodes > 1 and rng.random() < 0.7, hk * group, hk,
                         d, block, layout)
        w = work(case)
        # The plain forms pad a batch to its longest member: bounded too.
        pairs = case["B"] * case["HQ"] * _pad_pairs(case) if op in ("prompt", "tree") else 0
        rows = case["B"] * (case["hi"] + case["nodes"]) * hk * d if op == "tree" else 0
        if w["flops"] <= 4e12 and w["bytes"] <= 1.2e9 and pairs <= 1.7e10 and rows <= 1.2e9 and case.get("HQ", 1) <= 64:
            del case["name"]
            return case


def _pad_pairs(case):
    if case["op"] == "prompt":
        return case["hi"] * (case["hi"] + case["prefix"])
    return case["nodes"] * (case["hi"] + case["nodes"])


# --- what follows from a case alone ---------------------------------------

def _spread(tag, n, lo, hi):
    """n lengths in [lo, hi], spread over the logarithm, the longest among them."""
    rng = random.Random(f"{tag} {n} {lo} {hi}")
    out = [round((lo + 1) * ((hi + 1) / (lo + 1)) ** rng.random()) - 1 for _ in range(n)]
    out[rng.randrange(n)] = hi
    return out


def _prompt_lengths(case):
    q = _spread("prompt", case["B"], case["lo"], case["hi"])
    pre = _spread("prefix", case["B"], 0, case["prefix"]) if case["prefix"] else [0] * case["B"]
    return q, [a + b for a, b in zip(q, pre)]


def _tree_nodes(case):
    """Per request its nodes' parents (-1: a root).  A chain without a tree."""
    rng = random.Random(f"tree {case['B']} {case['nodes']}")
    if not case["tree"]:
        return [[i - 1 for i in range(case["nodes"])] for _ in range(case["B"])]
    sizes = [rng.randint(max(1, case["nodes"] // 3), case["nodes"]) for _ in range(case["B"])]
    sizes[-1] = case["nodes"]
    return [[-1 if i == 0 else rng.randint(max(0, i - 8), i - 1) for i in range(n)] for n in sizes]


def _ancestors(parents):
    """Per node the set of nodes it reads, itself among them, as an integer of bits."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return bits


def _valid_pairs(lq, lk, causal):
    if not causal:
        return lq * lk
    full = min(lq, lk)  # the last `full` rows read lk - full + 1 .. lk keys
    return full * (lk - full) + full * (full + 1) // 2


def work(case):
    op = case["op"]
    if op == "slots":
        have = _spread("have", case["B"], case["lo"], case["hi"])
        new = _spread("new", case["B"], case["new_lo"], case["new_hi"])
        s = case["block"]
        fresh = sum(-(-(h + n) // s) - -(-h // s) for h, n in zip(have, new))
        return {"bytes": 12 * case["B"] + 16 * (sum(new) + case["pad"]) + 8 * fresh, "flops": 0}
    D, HK = case["D"], case["HK"]
    if op == "write":
        return {"bytes": 8 * case["T"] * HK * D + 8 * (case["T"] + case["pad"]), "flops": 0}
    HQ = case["HQ"]
    if op == "prompt":
        lq, lk = _prompt_lengths(case)
        pairs = sum(_valid_pairs(a, b, case["causal"]) for a, b in zip(lq, lk))
        return {"bytes": 4 * HQ * D * sum(lq) + 4 * HK * D * sum(lk) + 4 * HQ * sum(lq),
                "flops": 4 * HQ * D * pairs}
    ctx = _spread("context", case["B"], case["lo"], case["hi"])
    trees = _tree_nodes(case)
    nodes = sum(map(len, trees))
    pairs = sum(c * len(t) + sum(b.bit_count() if hasattr(b, "bit_count") else bin(b).count("1") for b in _ancestors(t))
                for c, t in zip(ctx, trees))
    return {"bytes": 4 * HK * D * (sum(ctx) + nodes) + 4 * HQ * D * nodes + 4 * HQ * nodes
            + sum(4 * -(-(c + len(t)) // case["block"]) for c, t in zip(ctx, trees)),
            "flops": 4 * HQ * D * pairs}


# --- inputs -----------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _cu(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return _ints(out)


def _cache(gen, case, blocks):
    """K and V caches as (block, token, head, dim) views of either storage order."""
    shape = (blocks, case["block"], case["HK"], case["D"])
    if case["layout"] == "bhsd":
        shape = (shape[0], shape[2], shape[1], shape[3])
    kv = [torch.randn(shape, generator=gen, device="cuda", dtype=TORCH[case["dtype"]]) for _ in range(2)]
    return [t.transpose(1, 2) if case["layout"] == "bhsd" else t for t in kv]


def _table(gen, lengths, block, spare, width=None):
    """A table of shuffled block ids covering `lengths` tokens per row (0 elsewhere), and the ids left over."""
    used = [-(-n // block) for n in lengths]
    total = sum(used) + spare
    ids = torch.randperm(total, generator=gen, device="cuda").int()
    width = width or max(1, max(used))
    cols = torch.arange(width, device="cuda")
    n = _ints(used).long()
    first = torch.cumsum(n, 0) - n
    inside = cols[None, :] < n[:, None]
    at = (first[:, None] + cols[None, :]).clamp_(max=total - 1)
    return torch.where(inside, ids[at], 0).int().contiguous(), ids[sum(used):].contiguous(), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "slots":
        have = _spread("have", case["B"], case["lo"], case["hi"])
        new = _spread("new", case["B"], case["new_lo"], case["new_hi"])
        block = case["block"]
        after = [-(-(h + n) // block) for h, n in zip(have, new)]
        spare = sum(after) + case["B"]
        s["table"], s["free"], _ = _table(gen, have, block, spare, width=max(1, max(after)) + 1)
        s.update(lengths=_ints(have), counts=_ints(new), tokens=sum(new) + case["pad"])
        return s
    dtype = TORCH[case["dtype"]]
    HK, D = case["HK"], case["D"]
    if op == "write":
        T, pad = case["T"], case["pad"]
        blocks = -(-T // case["block"]) * 2 + 1
        s["k_cache"], s["v_cache"] = _cache(gen, case, blocks)
        qkv = torch.randn(T + pad, 2 * HK, D, generator=gen, device="cuda", dtype=dtype)
        s["k"], s["v"] = qkv[:, :HK], qkv[:, HK:]
        # Runs of a block's consecutive slots, the blocks in shuffled order.
        ids = torch.randperm(blocks, generator=gen, device="cuda")
        t = torch.arange(T, device="cuda")
        s["slots"] = torch.cat([ids[t // case["block"]] * case["block"] + t % case["block"],
                                torch.full((pad,), -1, dtype=torch.int64, device="cuda")])
        return s
    HQ = case["HQ"]
    s["scale"] = D**-0.5
    if op == "prompt":
        lq, lk = _prompt_lengths(case)
        same = lq == lk
        if case["packed"] and same:
            qkv = torch.randn(sum(lq), HQ + 2 * HK, D, generator=gen, device="cuda", dtype=dtype)
            s["q"], s["k"], s["v"] = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
        else:
            s["q"] = torch.randn(sum(lq), HQ, D, generator=gen, device="cuda", dtype=dtype)
            s["k"], s["v"] = (torch.randn(sum(lk), HK, D, generator=gen, device="cuda", dtype=dtype) for _ in range(2))
        s.update(cu_q=_cu(lq), cu_k=None if same else _cu(lk), max_q=max(lq), max_k=max(lk))
    else:
        ctx = _spread("context", case["B"], case["lo"], case["hi"])
        trees = _tree_nodes(case)
        total = [c + len(t) for c, t in zip(ctx, trees)]
        s["table"], _, blocks = _table(gen, total, case["block"], 3)
        s["k_cache"], s["v_cache"] = _cache(gen, case, blocks)
        nodes = sum(map(len, trees))
        s["q"] = torch.randn(nodes, HQ, D, generator=gen, device="cuda", dtype=dtype)
        s.update(lengths=_ints(ctx), cu_q=_cu(list(map(len, trees))), max_q=case["nodes"], max_k=max(total))
        s["mask"] = None
        if case["tree"]:
            words = -(-case["nodes"] // 64)
            rows = [[_signed(b >> 64 * w) for w in range(words)] for t in trees for b in _ancestors(t)]
            s["mask"] = _ints(rows, torch.int64)
    s["lse"] = torch.empty(HQ, s["q"].shape[0], device="cuda")
    return s


def _signed(bits):
    bits &= (1 << 64) - 1
    return bits - (1 << 64) if bits >> 63 else bits


# --- one pass ---------------------------------------------------------------

def run(s):
    return {"slots": _run_slots, "write": _run_write, "prompt": _run_prompt, "tree": _run_tree}[s["case"]["op"]](s)


def _run_slots(s):
    block, T = s["case"]["block"], s["tokens"]
    if own:
        from gfx950_gluon_tutorials_amd.attention import assign_slots
        r = assign_slots(s["lengths"], s["counts"], s["table"], s["free"], block, T)
        return {"cu": r.cu_seqlens, "slots": r.slots, "positions": r.positions, "taken": r.taken, "table": s["table"]}
    have, new, table, free = s["lengths"].long(), s["counts"].long(), s["table"], s["free"]
    B, W = table.shape
    end = torch.cumsum(new, 0)
    first = (have + block - 1) // block
    need = ((have + new + block - 1) // block).clamp(max=W) - first
    base = torch.cumsum(need, 0) - need
    tok = torch.arange(T, device=have.device)
    b = torch.searchsorted(end, tok, right=True).clamp(max=B - 1)
    real = tok < end[-1]
    pos = have[b] + tok - (end - new)[b]
    j = pos // block
    fresh = base[b] + j - first[b]
    ids = torch.where(j < first[b], table[b, j.clamp(max=W - 1)].long(), free[fresh.clamp(0, free.numel() - 1)].long())
    slots = torch.where(real & (j < W) & ((j < first[b]) | (fresh < free.numel())), ids * block + pos % block, -1)
    col = torch.arange(W, device=have.device)
    place = base[:, None] + col - first[:, None]
    added = (col >= first[:, None]) & (col < (first + need)[:, None])
    got = torch.where(place < free.numel(), free[place.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(added, got, table))
    cu = torch.cat([end.new_zeros(1), end]).int()
    return {"cu": cu, "slots": slots, "positions": torch.where(real, pos, 0), "taken": need.sum().int().reshape(1),
            "table": table}


def _run_write(s):
    k, v, kc, vc, slots = s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"]
    if own:
        from gfx950_gluon_tutorials_amd.attention import write_cache
        write_cache(k, v, kc, vc, slots)
        return {"k_cache": kc, "v_cache": vc}
    block = s["case"]["block"]
    # Rows without a slot repeat the first row that has one.
    real = slots >= 0
    row = torch.where(real, torch.arange(slots.numel(), device=slots.device), real.to(torch.int8).argmax())
    at = slots[row]
    kc[at // block, at % block] = k[row]
    vc[at // block, at % block] = v[row]
    return {"k_cache": kc, "v_cache": vc}


def _softmax_product(q, k, v, allowed, scale, group):
    """softmax(scale q k^T) v and the log-sum-exp, in the inputs' precision, over the allowed keys: q
    (B, Lq, HK * group, D), k and v (B, Lk, HK, D), allowed (B, Lq, Lk).  A few key/value heads at a time."""
    B, Lq, HQ, D = q.shape
    Lk, HK = k.shape[1], k.shape[2]
    out, lse = torch.empty_like(q), q.new_empty(B, HQ, Lq)
    bias = torch.zeros(allowed.shape, dtype=q.dtype, device=q.device).masked_fill_(~allowed, float("-inf"))
    step = max(1, min(HK, int(2**31 // (B * group * Lq * Lk))))
    for h in range(0, HK, step):
        n = min(step, HK - h)
        qh = q[:, :, h * group:(h + n) * group].reshape(B, Lq, n, group, D).permute(0, 2, 3, 1, 4)
        qh = qh.reshape(B, n, group * Lq, D)
        kh = k[:, :, h:h + n].permute(0, 2, 3, 1).contiguous()
        x = torch.matmul(qh, kh).reshape(B, n, group, Lq, Lk)
        x.mul_(scale).add_(bias[:, None, None])
        top = x.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), 0.0, top)
        x.sub_(top).exp_()
        total = x.sum(-1, keepdim=True)
        vh = v[:, :, h:h + n].permute(0, 2, 1, 3).contiguous()
        o = torch.matmul(x.reshape(B, n, group * Lq, Lk), vh).reshape(B, n, group, Lq, D)
        o = o / torch.where(total == 0, 1.0, total)
        out[:, :, h * group:(h + n) * group] = o.permute(0, 3, 1, 2, 4).reshape(B, Lq, n * group, D)
        lse[:, h * group:(h + n) * group] = (top + total.log()).reshape(B, n * group, Lq)
    return out, lse


def _pad(x, cu, longest, dtype):
    """(B, longest, ...) of packed rows, zeros behind each sequence, and the rows' places."""
    t = torch.arange(x.shape[0], device=x.device)
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    i = t - cu.long()[b]
    out = torch.zeros((cu.numel() - 1, longest) + tuple(x.shape[1:]), dtype=dtype, device=x.device)
    out[b, i] = x.to(dtype)
    return out, b, i


def _prompt_in(s, dtype):
    cu_k = s["cu_q"] if s["cu_k"] is None else s["cu_k"]
    q, b, i = _pad(s["q"], s["cu_q"], s["max_q"], dtype)
    k, _, _ = _pad(s["k"], cu_k, s["max_k"], dtype)
    v, _, _ = _pad(s["v"], cu_k, s["max_k"], dtype)
    lq, lk = (c[1:] - c[:-1] for c in (s["cu_q"], cu_k))
    rows, cols = torch.arange(s["max_q"], device=q.device), torch.arange(s["max_k"], device=q.device)
    allowed = (cols < lk[:, None])[:, None, :].expand(-1, s["max_q"], -1)
    if s["case"]["causal"]:
        allowed = allowed & (cols[None, None, :] <= rows[None, :, None] + (lk - lq)[:, None, None])
    o, lse = _softmax_product(q, k, v, allowed, s["scale"], s["case"]["HQ"] // s["case"]["HK"])
    return o[b, i], lse.transpose(1, 2)[b, i].t()


def _run_prompt(s):
    if own:
        from gfx950_gluon_tutorials_amd.attention import varlen_attention
        o = varlen_attention(s["q"], s["k"], s["v"], s["cu_q"], cu_seqlens_k=s["cu_k"], causal=s["case"]["causal"],
                             sm_scale=s["scale"], lse=s["lse"])
        return {"o": o, "lse": s["lse"]}
    o, lse = _prompt_in(s, torch.float32)
    return {"o": o.to(s["q"].dtype), "lse": lse.contiguous()}


def _tree_in(s, dtype):
    block = s["case"]["block"]
    q, b, i = _pad(s["q"], s["cu_q"], s["max_q"], dtype)
    pos = torch.arange(s["max_k"], device=q.device)
    ids = s["table"][:, pos // block].long()
    k, v = (c[ids, pos % block].to(dtype) for c in (s["k_cache"], s["v_cache"]))
    n = s["cu_q"][1:] - s["cu_q"][:-1]
    past = pos[None, :] - s["lengths"][:, None].long()  # the key's node, negative in the context
    node = past.clamp(min=0)[:, None, :].expand(-1, s["max_q"], -1)
    if s["mask"] is None:
        reads = node <= torch.arange(s["max_q"], device=q.device)[None, :, None]
    else:
        words = torch.zeros(q.shape[0], s["max_q"], s["mask"].shape[1], dtype=torch.int64, device=q.device)
        words[b, i] = s["mask"]
        word = torch.gather(words, 2, (node // 64).clamp(max=words.shape[2] - 1))
        reads = ((word >> (node % 64)) & 1).bool()
    allowed = (past < 0)[:, None, :] | (reads & (past < n[:, None])[:, None, :])
    o, lse = _softmax_product(q, k, v, allowed, s["scale"], s["case"]["HQ"] // s["case"]["HK"])
    return o[b, i], lse.transpose(1, 2)[b, i].t()


def _run_tree(s):
    if own:
        from gfx950_gluon_tutorials_amd.attention import tree_attention
        o = tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["cu_q"], s["mask"],
                           sm_scale=s["scale"], lse=s["lse"])
        return {"o": o, "lse": s["lse"]}
    o, lse = _tree_in(s, torch.float32)
    return {"o": o.to(s["q"].dtype), "lse": lse.contiguous()}


# --- the definition in 64 bits ------------------------------------------------

def exact(case, seed):
    """One sequence and one key/value head at a time, from the definition: for every row the allowed keys' scores,
    their largest, the exponentials' sum, the weighted values."""
    if case["op"] == "slots":
        return None
    s = prepare(case, seed)
    if case["op"] == "write":
        at = s["slots"][s["slots"] >= 0]
        page = torch.div(at, case["block"], rounding_mode="floor")
        out = {}
        for name, rows in (("k_cache", s["k"]), ("v_cache", s["v"])):
            out[name] = s[name].double()
            out[name][page, at - page * case["block"]] = rows[: at.numel()].double()
        return out
    group = case["HQ"] // case["HK"]
    ends = s["cu_q"].tolist()
    key_ends = (s["cu_q"] if s.get("cu_k") is None else s["cu_k"]).tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((case["HQ"], s["q"].shape[0]), float("-inf"), dtype=torch.float64, device="cuda")
    trees = _tree_nodes(case) if case["op"] == "tree" else None
    for b in range(case["B"]):
        r0, r1 = ends[b], ends[b + 1]
        if case["op"] == "prompt":
            k0, k1 = key_ends[b], key_ends[b + 1]
            keys, values = s["k"][k0:k1], s["v"][k0:k1]
            shift = (k1 - k0) - (r1 - r0)
        else:
            context = int(s["lengths"][b])
            at = torch.arange(context + r1 - r0, device="cuda")
            page = s["table"][b].long()[at // case["block"]]
            keys, values = (c[page, at % case["block"]] for c in (s["k_cache"], s["v_cache"]))
            sees = torch.zeros(r1 - r0, r1 - r0, dtype=torch.bool)
            for i, p in enumerate(trees[b]):
                if p >= 0:
                    sees[i] = sees[p]
                sees[i, i] = True
            sees = sees.cuda()
        if r1 == r0 or len(keys) == 0:
            continue
        for g in range(case["HK"]):
            kk, vv = keys[:, g].double(), values[:, g].double()
            for h in range(g * group, (g + 1) * group):
                x = (s["q"][r0:r1, h].double() @ kk.t().contiguous()) * s["scale"]
                if case["op"] == "tree":
                    x[:, context:][~sees] = float("-inf")
                elif case["causal"]:
                    late = torch.arange(len(keys), device="cuda")[None] > torch.arange(r1 - r0, device="cuda")[:, None] + shift
                    x.masked_fill_(late, float("-inf"))
                top = x.max(dim=1, keepdim=True).values.clamp(min=-1e300)
                w = (x - top).exp()
                z = w.sum(dim=1, keepdim=True)
                out[r0:r1, h] = (w @ vv) / z.clamp(min=1e-300)
                lse[h, r0:r1] = (top + z.log())[:, 0]
    return {"o": out, "lse": lse}
