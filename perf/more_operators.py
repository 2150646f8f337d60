"""The operators of serving with latent attention, as workloads: cases, inputs,
the plain form of each, and the calls a user's program makes of them.

* ``rotary``: rotary positions into packed rows (``rotary``).
* ``write``: one latent vector and one rotated key a token, normalised, rotated
  and written into a paged cache (``write_latent``).
* ``decode``: attention over that cache, keys and values absorbed into the
  queries (``latent_attention``): single tokens, chains and trees.
* ``prompt``: attention over packed prompts whose keys and values were expanded
  from the latents (``latent_varlen_attention``).

The lengths of a batch and the shape of a draft tree follow from the case
alone, so its work is known without its inputs; block ids, positions and values
come from the seed.  Caches hold more blocks than the batch uses, in shuffled
order.
"""

import math
import random

import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}
RANK, ROPE, NOPE, VALUE = 512, 64, 128, 128  # a latent, its rotated key; a head's key and value
EPS = 1e-6


def _rotary(name, dtype, T, H, spare, D, first, dim, interleaved=False, inverse=False, factor=1.0):
    return {"name": name, "op": "rotary", "dtype": dtype, "T": T, "H": H, "spare": spare, "D": D, "first": first,
            "dim": dim, "interleaved": interleaved, "inverse": inverse, "factor": factor}


def _write(name, dtype, T, block, pad=0, outputs=False, interleaved=True):
    return {"name": name, "op": "write", "dtype": dtype, "T": T, "block": block, "pad": pad, "outputs": outputs,
            "interleaved": interleaved}


def _decode(name, dtype, B, lo, hi, nodes, tree, H, block):
    return {"name": name, "op": "decode", "dtype": dtype, "B": B, "lo": lo, "hi": hi, "nodes": nodes, "tree": tree,
            "H": H, "block": block}


def _prompt(name, dtype, B, lo, hi, H, prefix=0, causal=True):
    return {"name": name, "op": "prompt", "dtype": dtype, "B": B, "lo": lo, "hi": hi, "H": H, "prefix": prefix,
            "causal": causal}


def listed():
    return [
        # One decoding step of 64 requests: the queries and keys of one fused q/k/v projection, in one call.
        _rotary("rotary_bf16_t64", "bf16", 64, 40, 8, 128, 0, 128),
        # A batch of prompts' queries and keys, one layer.
        _rotary("rotary_bf16_t16384", "bf16", 16384, 40, 8, 128, 0, 128),
        # The gradient of latent queries' last 64 values, neighbouring pairs, positions scaled for long contexts.
        _rotary("rotary_f16_t4001_part", "f16", 4001, 32, 0, 192, 128, 64, True, True, factor=16.0),
        # One decoding step's latents, one layer: latency.
        _write("write_bf16_t64", "bf16", 64, 16),
        # A batch of prompts' latents, which the expansion reads too.
        _write("write_bf16_t16384", "bf16", 16384, 64, pad=37, outputs=True),
        # One user, a short conversation, one GPU's heads of 8: latency.
        _decode("decode_bf16_b1_s700_h16", "bf16", 1, 700, 700, 1, False, 16, 64),
        # A serving batch, one token per request, uneven contexts, one GPU's heads of 8.
        _decode("decode_bf16_b64_s8192_h16", "bf16", 64, 100, 8192, 1, False, 16, 64),
        # The same with all heads on one GPU (heads not split).
        _decode("decode_bf16_b64_s8192_h128", "bf16", 64, 100, 8192, 1, False, 128, 64),
        # Verification of drafted trees of up to 12 nodes for 16 requests.
        _decode("tree_f16_b16_n12_h32", "f16", 16, 500, 12000, 12, True, 32, 32),
        # A single short prompt: latency.
        _prompt("prompt_bf16_1x197_h16", "bf16", 1, 197, 197, 16),
        # Uneven chunks of prompts behind cached prefixes.
        _prompt("prompt_f16_12x100_2500_h32", "f16", 12, 100, 2500, 32, prefix=1500),
        # One long prompt: the largest product.
        _prompt("prompt_bf16_1x16384_h32", "bf16", 1, 16384, 16384, 32),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "write", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    while True:
        dtype, block = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
        H = rng.choice([1, 4, 8, 16, 20, 32, 64, 128])
        if op == "rotary":
            D = rng.choice([64, 80, 96, 128, 192, 256])
            first, dim = rng.choice([(0, D), (0, 32), (0, 64), (D - 64, 64), (D - 48, 48)])
            case = _rotary("", dtype, _log(rng, 1, 16384), rng.choice([H, 5, 40, 72]), rng.choice([0, 0, 1, 8]), D, first,
                           dim, rng.random() < 0.5, rng.random() < 0.3, rng.choice([1.0, 1.0, 4.0, 40.0]))
        elif op == "write":
            case = _write("", dtype, _log(rng, 1, 16384), block, rng.choice([0, 0, _log(rng, 1, 100)]),
                          rng.random() < 0.5, rng.random() < 0.5)
        elif op == "decode":
            lo = _log(rng, 1, 32768) - 1
            hi = rng.choice([lo, _log(rng, lo + 1, 131072)])
            nodes = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 2, 70)])
            case = _decode("", dtype, _log(rng, 1, 128), lo, hi, nodes, nodes > 1 and rng.random() < 0.6, H, block)
        else:
            lo = _log(rng, 1, 8192)
            hi = rng.choice([lo, _log(rng, lo, 16384)])
            case = _prompt("", dtype, _log(rng, 1, 64), lo, hi, H, prefix=rng.choice([0, 0, _log(rng, 1, 4096)]),
                           causal=rng.random() < 0.8)
        w = work(case)
        # The plain forms pad a batch to its longest member: bounded too.
        pairs = rows = 0
        if op == "decode":
            rows = case["B"] * (hi + nodes)
            pairs = rows * H * nodes
        elif op == "prompt":
            rows = case["B"] * (hi + case["prefix"]) * H
            pairs = case["B"] * H * hi * (hi + case["prefix"])
        if w["flops"] <= 2.7e12 and w["bytes"] <= 6e8 and pairs <= 8.6e9 and rows <= 2e6:
            del case["name"]
            return case


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
    if op == "rotary":
        return {"bytes": case["T"] * (4 * case["H"] * case["D"] + 8) + 4 * case["dim"],
                "flops": 3 * case["T"] * case["H"] * case["dim"]}
    if op == "write":
        rows = case["T"] + case["pad"]
        return {"bytes": 2 * (RANK + ROPE) * (case["T"] + rows * (2 if case["outputs"] else 1)) + 16 * rows + 2 * RANK
                + 4 * ROPE, "flops": rows * (4 * RANK + 3 * ROPE)}
    H = case["H"]
    if op == "prompt":
        lq, lk = _prompt_lengths(case)
        pairs = sum(_valid_pairs(a, b, case["causal"]) for a, b in zip(lq, lk))
        return {"bytes": 2 * H * (NOPE + ROPE + VALUE) * sum(lq) + 2 * (H * (NOPE + VALUE) + ROPE) * sum(lk)
                + 4 * H * sum(lq), "flops": 2 * H * (NOPE + ROPE + VALUE) * pairs}
    ctx = _spread("context", case["B"], case["lo"], case["hi"])
    trees = _tree_nodes(case)
    nodes = sum(map(len, trees))
    pairs = sum(c * len(t) + sum(bin(b).count("1") for b in _ancestors(t)) for c, t in zip(ctx, trees))
    return {"bytes": 2 * (RANK + ROPE) * (sum(ctx) + nodes) + 2 * H * (RANK + ROPE + RANK) * nodes + 4 * H * nodes
            + sum(4 * -(-(c + len(t)) // case["block"]) for c, t in zip(ctx, trees)),
            "flops": 2 * H * (RANK + ROPE + RANK) * pairs}


# --- inputs -----------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _cu(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return _ints(out)


def _frequencies(dim, factor):
    """Radians a position, 64 bits: base 10000; with a factor the pairs that turn less than 4 times over 4096 positions
    are slowed by it, those that turn more than 32 times kept, and a ramp between."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = 10000.0 ** (-2 * i / dim)
    keep = ((4096 * f / (2 * math.pi) - 4) / 28).clamp(0, 1)
    return (f * (keep + (1 - keep) / factor)).cuda()


def _positions(gen, rows):
    """Runs of consecutive positions, as a batch of chunks has them."""
    t = torch.arange(rows, device="cuda")
    chunk = max(1, rows // 64)
    start = torch.randint(0, 131072, (rows // chunk + 1,), generator=gen, device="cuda")
    return start[t // chunk] + t % chunk


def _table(gen, lengths, block, spare):
    """A table of shuffled block ids covering `lengths` tokens per row (0 elsewhere)."""
    used = [-(-n // block) for n in lengths]
    total = sum(used) + spare
    ids = torch.randperm(total, generator=gen, device="cuda").int()
    cols = torch.arange(max(1, max(used)), device="cuda")
    n = _ints(used).long()
    first = torch.cumsum(n, 0) - n
    at = (first[:, None] + cols[None, :]).clamp_(max=total - 1)
    return torch.where(cols[None, :] < n[:, None], ids[at], 0).int().contiguous(), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], TORCH[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    s = {"case": case}
    if op == "rotary":
        s["x"] = randn(case["T"], case["H"] + case["spare"], case["D"])[:, :case["H"]]
        s["positions"] = _positions(gen, case["T"])
        s["freqs"] = _frequencies(case["dim"], case["factor"])
        s["scale"] = 0.1 * math.log(case["factor"]) + 1.0
        return s
    if op == "write":
        T, rows = case["T"], case["T"] + case["pad"]
        blocks = -(-T // case["block"]) * 2 + 1
        s["cache"] = randn(blocks, case["block"], RANK + ROPE)
        down = randn(rows, RANK + ROPE)  # one projection makes both
        s["c"], s["k_rope"] = down[:, :RANK], down[:, RANK:]
        s["weight"] = (1 + 0.2 * torch.randn(RANK, generator=gen, device="cuda")).to(dtype)
        s["positions"], s["freqs"] = _positions(gen, rows), _frequencies(ROPE, 1.0)
        ids = torch.randperm(blocks, generator=gen, device="cuda")
        t = torch.arange(T, device="cuda")
        s["slots"] = torch.cat([ids[t // case["block"]] * case["block"] + t % case["block"],
                                torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")])
        s["c_out"] = torch.empty(rows, RANK, dtype=dtype, device="cuda") if case["outputs"] else None
        s["k_out"] = torch.empty(rows, ROPE, dtype=dtype, device="cuda") if case["outputs"] else None
        return s
    H = case["H"]
    s["scale"] = (NOPE + ROPE) ** -0.5
    if op == "prompt":
        lq, lk = _prompt_lengths(case)
        same = lq == lk
        s["q"] = randn(sum(lq), H, NOPE + ROPE)
        kv = randn(sum(lk), H, NOPE + VALUE)  # the latents' expansion
        s["k"], s["v"], s["k_rope"] = kv[..., :NOPE], kv[..., NOPE:], randn(sum(lk), ROPE)
        s.update(cu_q=_cu(lq), cu_k=None if same else _cu(lk), max_q=max(lq), max_k=max(lk))
    else:
        ctx = _spread("context", case["B"], case["lo"], case["hi"])
        trees = _tree_nodes(case)
        total = [c + len(t) for c, t in zip(ctx, trees)]
        s["table"], blocks = _table(gen, total, case["block"], 3)
        s["cache"] = randn(blocks, case["block"], RANK + ROPE)
        # Scores of a spread like a prompt's: the absorbed query's length goes with the root of its head's key.
        s["q"] = randn(sum(map(len, trees)), H, RANK + ROPE).mul_(((NOPE + ROPE) / (RANK + ROPE)) ** 0.5)
        s.update(lengths=_ints(ctx), cu_q=_cu(list(map(len, trees))), max_q=case["nodes"], max_k=max(total), mask=None)
        if case["tree"]:
            words = -(-case["nodes"] // 64)
            rows = [[_signed(b >> 64 * w) for w in range(words)] for t in trees for b in _ancestors(t)]
            s["mask"] = _ints(rows, torch.int64)
    s["lse"] = torch.empty(H, s["q"].shape[0], device="cuda")
    return s


def _signed(bits):
    bits &= (1 << 64) - 1
    return bits - (1 << 64) if bits >> 63 else bits


# --- one pass ---------------------------------------------------------------

def run(s):
    return {"rotary": _run_rotary, "write": _run_write, "decode": _run_decode, "prompt": _run_prompt}[s["case"]["op"]](s)


def _rotate(x, positions, freqs, interleaved, inverse, scale):
    """The pairs of x (rows, heads, dim), fp32, turned by positions * freqs; the angles in 64 bits."""
    t = positions.double()[:, None] * freqs
    cos, sin = (t.cos() * scale).float()[:, None], ((-t if inverse else t).sin() * scale).float()[:, None]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _run_rotary(s):
    c = s["case"]
    if own:
        from gfx950_gluon_tutorials_amd.attention import rotary
        return rotary(s["x"], s["positions"], s["freqs"], first=c["first"], interleaved=c["interleaved"],
                      inverse=c["inverse"], scale=s["scale"])
    x, end = s["x"], c["first"] + c["dim"]
    y = _rotate(x[..., c["first"]:end].float(), s["positions"], s["freqs"], c["interleaved"], c["inverse"], s["scale"])
    return torch.cat((x[..., :c["first"]], y.to(x.dtype), x[..., end:]), -1)


def _run_write(s):
    c, k, cache, slots, interleaved = s["c"], s["k_rope"], s["cache"], s["slots"], s["case"]["interleaved"]
    if own:
        from gfx950_gluon_tutorials_amd.attention import write_latent
        write_latent(c, k, cache, slots, weight=s["weight"], eps=EPS, positions=s["positions"], freqs=s["freqs"],
                     interleaved=interleaved, c_out=s["c_out"], k_out=s["k_out"])
        return {"cache": cache, "c": s["c_out"], "k": s["k_out"]} if s["c_out"] is not None else {"cache": cache}
    x = c.float()
    y = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()).to(c.dtype)
    z = _rotate(k.float()[:, None], s["positions"], s["freqs"], interleaved, False, 1.0)[:, 0].to(k.dtype)
    # Rows without a slot repeat the first row that has one.
    real = slots >= 0
    row = torch.where(real, torch.arange(slots.numel(), device=slots.device), real.to(torch.int8).argmax())
    at = slots[row]
    cache[at // s["case"]["block"], at % s["case"]["block"]] = torch.cat((y, z), -1)[row]
    if s["c_out"] is None:
        return {"cache": cache}
    s["c_out"].copy_(y)
    s["k_out"].copy_(z)
    return {"cache": cache, "c": s["c_out"], "k": s["k_out"]}


def _softmax_product(q, k, v, allowed, scale):
    """softmax(scale q k^T) v and the log-sum-exp in fp32 over the allowed keys: q (B, H, Lq, DK), k (B, H or 1, Lk, DK),
    v (B, H or 1, Lk, DV), allowed (B, Lq, Lk).  A few sequences and heads at a time."""
    B, H, Lq, _ = q.shape
    Lk, shared = k.shape[2], k.shape[1] == 1
    out, lse = q.new_empty(B, H, Lq, v.shape[3]), q.new_empty(B, H, Lq)
    bias = torch.zeros(allowed.shape, dtype=q.dtype, device=q.device).masked_fill_(~allowed, float("-inf"))
    nh = max(1, min(H, 2**31 // max(1, Lq * Lk)))
    nb = max(1, 2**31 // max(1, nh * Lq * Lk))
    for b in range(0, B, nb):
        for h in range(0, H, nh):
            part, keys = (slice(b, b + nb), slice(h, h + nh)), (slice(b, b + nb), slice(0, 1) if shared else slice(h, h + nh))
            qp, kp, vp = q[part], k[keys].transpose(2, 3).contiguous(), v[keys].contiguous()
            n, m = qp.shape[:2]
            if shared:
                x = torch.matmul(qp.reshape(n, m * Lq, -1), kp[:, 0]).reshape(n, m, Lq, Lk)
            else:
                x = torch.matmul(qp, kp)
            x.mul_(scale).add_(bias[part[0], None])
            top = x.amax(-1, keepdim=True)
            top = torch.where(top == float("-inf"), 0.0, top)
            x.sub_(top).exp_()
            total = x.sum(-1, keepdim=True)
            if shared:
                o = torch.matmul(x.reshape(n, m * Lq, Lk), vp[:, 0]).reshape(n, m, Lq, -1)
            else:
                o = torch.matmul(x, vp)
            out[part] = o / torch.where(total == 0, 1.0, total)
            lse[part] = (top + total.log())[..., 0]
    return out, lse


def _pad(x, cu, longest):
    """(B, longest, ...) of packed rows in fp32, zeros behind each sequence, and the rows' places."""
    t = torch.arange(x.shape[0], device=x.device)
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    i = t - cu.long()[b]
    out = torch.zeros((cu.numel() - 1, longest) + tuple(x.shape[1:]), device=x.device)
    out[b, i] = x.float()
    return out, b, i


def _run_prompt(s):
    causal = s["case"]["causal"]
    if own:
        from gfx950_gluon_tutorials_amd.attention import latent_varlen_attention
        o = latent_varlen_attention(s["q"], s["k"], s["v"], s["k_rope"], s["cu_q"], cu_seqlens_k=s["cu_k"],
                                    causal=causal, sm_scale=s["scale"], lse=s["lse"])
        return {"o": o, "lse": s["lse"]}
    cu_k = s["cu_q"] if s["cu_k"] is None else s["cu_k"]
    q, b, i = _pad(s["q"], s["cu_q"], s["max_q"])
    keys = torch.cat((s["k"], s["k_rope"][:, None].expand(-1, s["case"]["H"], -1)), -1)
    k, v = (_pad(x, cu_k, s["max_k"])[0].transpose(1, 2) for x in (keys, s["v"]))
    lq, lk = (c[1:] - c[:-1] for c in (s["cu_q"], cu_k))
    rows, cols = torch.arange(s["max_q"], device=q.device), torch.arange(s["max_k"], device=q.device)
    allowed = (cols < lk[:, None])[:, None, :].expand(-1, s["max_q"], -1)
    if causal:
        allowed = allowed & (cols[None, None, :] <= rows[None, :, None] + (lk - lq)[:, None, None])
    o, lse = _softmax_product(q.transpose(1, 2), k, v, allowed, s["scale"])
    return {"o": o.transpose(1, 2)[b, i].to(s["q"].dtype), "lse": lse.transpose(1, 2)[b, i].t().contiguous()}


def _run_decode(s):
    if own:
        from gfx950_gluon_tutorials_amd.attention import latent_attention
        o = latent_attention(s["q"], s["cache"], s["table"], s["lengths"], s["cu_q"], s["mask"], sm_scale=s["scale"],
                             lse=s["lse"])
        return {"o": o, "lse": s["lse"]}
    block = s["case"]["block"]
    q, b, i = _pad(s["q"], s["cu_q"], s["max_q"])
    pos = torch.arange(s["max_k"], device=q.device)
    rows = s["cache"][s["table"][:, pos // block].long(), pos % block].float()[:, None]
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
    o, lse = _softmax_product(q.transpose(1, 2), rows, rows[..., :RANK], allowed, s["scale"])
    return {"o": o.transpose(1, 2)[b, i].to(s["q"].dtype), "lse": lse.transpose(1, 2)[b, i].t().contiguous()}


# --- the definition in 64 bits ------------------------------------------------

def _turned(x, case, positions, freqs, scale):
    """The rotation as complex numbers: pair (a, b) as a + bi, times scale e^(i angle)."""
    x = x.double()
    half = x.shape[-1] // 2
    pairs = x.unflatten(-1, (half, 2)) if case["interleaved"] else x.unflatten(-1, (2, half)).transpose(-1, -2)
    angle = positions.double()[:, None] * freqs
    if case.get("inverse"):
        angle = -angle
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, scale), angle)[:, None])
    return (turned if case["interleaved"] else turned.transpose(-1, -2)).flatten(-2)


def exact(case, seed):
    """From the definitions.  The attentions one sequence at a time: for every row the allowed keys' scores, their
    largest, the exponentials' sum, the weighted values."""
    s = prepare(case, seed)
    if case["op"] == "rotary":
        out = s["x"].double()
        part = slice(case["first"], case["first"] + case["dim"])
        out[..., part] = _turned(s["x"][..., part], case, s["positions"], s["freqs"], s["scale"])
        return out
    if case["op"] == "write":
        c = s["c"].double()
        c = c / (c.pow(2).sum(-1, keepdim=True) / RANK + EPS).sqrt() * s["weight"].double()
        k = _turned(s["k_rope"][:, None], case, s["positions"], s["freqs"], 1.0)[:, 0]
        at = s["slots"][s["slots"] >= 0]
        page = torch.div(at, case["block"], rounding_mode="floor")
        cache = s["cache"].double()
        cache[page, at - page * case["block"]] = torch.cat((c, k), 1)[: at.numel()]
        return {"cache": cache, "c": c, "k": k} if case["outputs"] else {"cache": cache}
    H = case["H"]
    ends = s["cu_q"].tolist()
    key_ends = (s["cu_q"] if s.get("cu_k") is None else s["cu_k"]).tolist()
    width = RANK if case["op"] == "decode" else VALUE
    out = torch.zeros(ends[-1], H, width, dtype=torch.float64, device="cuda")
    lse = torch.full((H, ends[-1]), float("-inf"), dtype=torch.float64, device="cuda")
    trees = _tree_nodes(case) if case["op"] == "decode" else None
    for b in range(case["B"]):
        r0, r1 = ends[b], ends[b + 1]
        if case["op"] == "decode":
            context = int(s["lengths"][b])
            at = torch.arange(context + r1 - r0, device="cuda")
            latents = s["cache"][s["table"][b].long()[at // case["block"]], at % case["block"]].double()
            hidden = torch.zeros(r1 - r0, len(at), dtype=torch.bool)
            for i, p in enumerate(trees[b]):
                hidden[i, context:] = True if p < 0 else hidden[p, context:]
                hidden[i, context + i] = False
        else:
            k0, k1 = key_ends[b], key_ends[b + 1]
            at = torch.arange(k1 - k0, device="cuda")
            hidden = None
            if case["causal"]:
                hidden = at[None] > torch.arange(r1 - r0, device="cuda")[:, None] + (k1 - k0) - (r1 - r0)
        if r1 == r0 or len(at) == 0:
            continue
        for h in range(H):
            if case["op"] == "decode":
                keys, values = latents, latents[:, :RANK]
            else:
                keys = torch.cat((s["k"][k0:k1, h], s["k_rope"][k0:k1]), 1).double()
                values = s["v"][k0:k1, h].double()
            x = (s["q"][r0:r1, h].double() @ keys.t().contiguous()) * s["scale"]
            if hidden is not None:
                x.masked_fill_(hidden.to(x.device), float("-inf"))
            top = x.max(dim=1, keepdim=True).values.clamp(min=-1e300)
            w = x.sub_(top).exp_()
            z = w.sum(dim=1, keepdim=True)
            out[r0:r1, h] = (w @ values) / z.clamp(min=1e-300)
            lse[h, r0:r1] = (top + z.log())[:, 0]
    return {"o": out, "lse": lse}
