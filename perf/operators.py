"""Work items of one speculative-decoding step over an 8-bit paged K/V cache.

Three operators, as a serving step runs them for each layer or once a step:

* ``append``    -- rotate the step's queries and keys by their positions and append
                   the keys and values to a paged cache of 8-bit codes with one
                   scale for each (block, KV head);
* ``attention`` -- attention of the step's packed queries (single tokens, drafted
                   tokens under verification, prompt chunks) over that cache;
* ``verify``    -- acceptance of drafted tokens against the target's probabilities
                   and the sample that follows, from given uniform numbers.

``run`` computes them in elementary torch operations, or (``own``) through the
package's entry points.  Cache: codes [num_blocks, kv_heads, block, head_size]
(int8, or float8_e4m3fn), scales float32 [num_blocks, kv_heads]; a code stands for
code * scale.
"""

import math
import random

import torch

own = False

_ACT = {"fp16": torch.float16, "bf16": torch.bfloat16}
_CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_TOP = {"int8": 127.0, "e4m3": 448.0}
_TINY = 2.0 ** -100  # a smaller scale is held as zero
_THETA = 1e6
_POSITIONS = 1 << 17  # rows of the rotation tables
_DEVICE = "cuda"


def _steps(op, name, geometry, act, code, block, requests, query, ctx, chunks=0, chunk=0, chunk_ctx=0):
    """A case of packed requests: ``requests`` of ``query`` tokens each with whole contexts in
    ``ctx``, then ``chunks`` prompt chunks of ``chunk`` tokens after ``chunk_ctx`` computed ones."""

    return {"op": op, "name": name, "hq": geometry[0], "hkv": geometry[1], "d": geometry[2], "act": act, "code": code,
            "block": block, "requests": requests, "query": query, "ctx_min": ctx[0], "ctx_max": ctx[1],
            "chunks": chunks, "chunk": chunk, "chunk_ctx": chunk_ctx}


def listed():
    return [
        # One user, one token, a short context: the latency of a single call.
        _steps("append", "append one token", (28, 4, 128), "fp16", "int8", 16, 1, 1, (201, 201)),
        # A decode batch of drafted tokens (one committed and four drafted each).
        _steps("append", "append drafts", (28, 4, 128), "bf16", "int8", 16, 64, 5, (512, 4096)),
        # Floating-point codes, small heads, larger blocks, odd lengths.
        _steps("append", "append ragged small heads", (14, 2, 64), "fp16", "e4m3", 32, 37, 3, (1, 1500), 3, 333, 77),
        # Prompt chunks of a long prefill.
        _steps("append", "append prompts", (40, 8, 128), "bf16", "int8", 16, 0, 1, (1, 1), 4, 2048, 2040),
        # One user, one token, a short context.
        _steps("attention", "attend one short", (28, 4, 128), "fp16", "int8", 16, 1, 1, (201, 201)),
        # The decode batch of the attention benchmark: 64 requests of 512 to 4096 tokens.
        _steps("attention", "attend decode batch", (28, 4, 128), "bf16", "int8", 16, 64, 1, (512, 4096)),
        # Few requests with long contexts: the work of one request is split over the GPU.
        _steps("attention", "attend long", (64, 8, 128), "fp16", "e4m3", 32, 3, 1, (20000, 65001)),
        # Verification of four drafts for each of 32 requests.
        _steps("attention", "attend drafts", (14, 2, 64), "fp16", "int8", 16, 32, 5, (300, 8000)),
        # A mixed step: one prompt chunk of 2048 tokens and 64 decodes.
        _steps("attention", "attend mixed", (40, 8, 128), "bf16", "int8", 16, 64, 1, (256, 8192), 1, 2048, 4096),
        # One user, four drafts from a draft model.
        {"op": "verify", "name": "verify one", "requests": 1, "drafts_min": 4, "drafts_max": 4, "vocab": 152064,
         "probs": True},
        # A batch with four drafts each.
        {"op": "verify", "name": "verify batch", "requests": 64, "drafts_min": 4, "drafts_max": 4, "vocab": 152064,
         "probs": True},
        # Drafts looked up in the context (no draft probabilities), ragged, some requests without any, an odd vocabulary.
        {"op": "verify", "name": "verify lookups", "requests": 150, "drafts_min": 0, "drafts_max": 7, "vocab": 50001,
         "probs": False},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""

    return _whole(max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))))))))


def _whole(n):
    return n + (n == 3 << 10)


def draw(rng):
    op = rng.choice(("append", "attention", "verify"))
    if op == "verify":
        vocab = _spread(rng, 1000, 152064)
        n = _spread(rng, 1, 64 if vocab > 60000 else 150)
        low = rng.randrange(0, 4)
        return {"op": op, "requests": n, "drafts_min": low, "drafts_max": low + rng.randrange(0, 5), "vocab": vocab,
                "probs": rng.random() < 0.6}
    hq, hkv, d = rng.choice(((14, 2, 64), (28, 4, 128), (12, 2, 128), (40, 8, 128), (64, 8, 128), (16, 16, 64), (16, 1, 128)))
    block = rng.choice((16, 16, 32, 64))
    act, code = rng.choice(("fp16", "bf16")), rng.choice(("int8", "int8", "e4m3"))
    if rng.random() < 0.3:  # prompt chunks, perhaps beside decodes
        chunk = _spread(rng, 17, 2048)
        case = _steps(op, "", (hq, hkv, d), act, code, block, rng.choice((0, 0, 5, 31)), 1, (16, _spread(rng, 17, 4096)),
                      1 if chunk > 700 else rng.randrange(1, 4), chunk, rng.choice((0, _whole(rng.randrange(0, 4096)))))
    else:
        n = _spread(rng, 1, 64)
        high = _spread(rng, 8, max(9, min(65000, 150000 // n // max(1, hkv // 4))))
        case = _steps(op, "", (hq, hkv, d), act, code, block, n, rng.choice((1, 1, 1, 2, 4, 5, 8)), (_spread(rng, 1, high), high))
    del case["name"]
    return case


def _requests(case):
    """[(computed, query tokens)] of a case of packed requests; the same for every seed."""

    rng = random.Random("%s/%s/%s" % (case["requests"], case["ctx_min"], case["ctx_max"]))
    got = []
    for _ in range(case["requests"]):
        ctx = _whole(rng.randint(case["ctx_min"], case["ctx_max"]))
        got.append((max(0, ctx - case["query"]), case["query"]))
    return got + [(case["chunk_ctx"], case["chunk"])] * case["chunks"]


def _drafts(case):
    rng = random.Random("%s/%s" % (case["requests"], case["vocab"]))
    return [rng.randint(case["drafts_min"], case["drafts_max"]) for _ in range(case["requests"])]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=_DEVICE)


def _quantise(x, code):
    """Codes and scales of x [blocks, heads, tokens, d], one scale for each block and head."""

    scale = x.abs().amax(dim=(2, 3)) / _TOP[code]
    y = x / scale[..., None, None]
    return (y.round() if code == "int8" else y).to(_CODE[code]), scale


def _pool(gen, blocks, case):
    """A cache's contents: normal values, a few strong channels in the keys, as in trained models."""

    shape = (blocks, case["hkv"], case["block"], case["d"])
    strong = torch.ones(case["d"], device=_DEVICE)
    strong[3::37] = 3.0
    keys, key_scales = _quantise(torch.randn(shape, device=_DEVICE, generator=gen) * strong, case["code"])
    values, value_scales = _quantise(torch.randn(shape, device=_DEVICE, generator=gen), case["code"])
    return keys, values, key_scales, value_scales


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE)
    gen.manual_seed(seed)
    return (_prepare_verify if case["op"] == "verify" else _prepare_step)(case, gen)


def _prepare_step(case, gen):
    reqs = _requests(case)
    hq, hkv, d, bs, act = case["hq"], case["hkv"], case["d"], case["block"], _ACT[case["act"]]
    n, queries = len(reqs), [q for _, q in reqs]
    need = [-(-(c + q) // bs) for c, q in reqs]
    starts = [0]
    for q in queries:
        starts.append(starts[-1] + q)
    total, stride = sum(need), max(need)
    blocks = total + 9
    order = torch.randperm(blocks, device=_DEVICE, generator=gen).to(torch.int32).cpu().tolist()
    rows, at = [], 0
    for k in need:
        rows.append(order[at:at + k] + [order[at]] * (stride - k))
        at += k
    keys, values, key_scales, value_scales = _pool(gen, blocks, case)
    state = {
        "op": case["op"], "case": case, "keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales,
        "tables": _ints(rows), "computed": _ints([c for c, _ in reqs]), "query_start": _ints(starts),
        "max_query": max(queries), "max_seq": max(c + q for c, q in reqs),
    }
    tokens = starts[-1]
    if case["op"] == "attention":
        state["query"] = (torch.randn((tokens, hq, d), device=_DEVICE, generator=gen) * 1.5).to(act)
        state["scale"] = 1.0 / math.sqrt(d)
        # The requests of one query token each, and the others: (requests, their longest query and context, the rows of
        # the batch, and each row's request within the group and place in it).
        state["groups"] = []
        for wanted in ([i for i in range(n) if queries[i] == 1], [i for i in range(n) if queries[i] != 1]):
            if wanted:
                at = [(starts[i] + j, k, j) for k, i in enumerate(wanted) for j in range(queries[i])]
                state["groups"].append((_ints(wanted, torch.long), max(queries[i] for i in wanted),
                                        max(sum(reqs[i]) for i in wanted)) + tuple(_ints(c, torch.long) for c in zip(*at)))
        return state
    width = (hq + 2 * hkv) * d
    state["qkv"] = torch.randn((tokens, width), device=_DEVICE, generator=gen).to(act)
    state["positions"] = _ints([c + j for c, q in reqs for j in range(q)])
    angle = torch.outer(torch.arange(_POSITIONS, device=_DEVICE, dtype=torch.float32),
                        1.0 / _THETA ** (torch.arange(0, d, 2, device=_DEVICE, dtype=torch.float32) / d)).repeat(1, 2)
    state["cos"], state["sin"] = angle.cos().to(act), angle.sin().to(act)
    # The blocks that the step writes to: (request, block of the request), and the pool's block.
    touched = [(r, b) for r, (c, q) in enumerate(reqs) for b in range(c // bs, -(-(c + q) // bs))]
    state["touched"] = tuple(_ints(v, torch.long) for v in zip(*touched))
    state["touched_blocks"] = _ints([rows[r][b] for r, b in touched])
    return state


def _prepare_verify(case, gen):
    drafts, vocab = _drafts(case), case["vocab"]
    starts = [0]
    for k in drafts:
        starts.append(starts[-1] + k + 1)
    total = sum(drafts)
    # A target's logits, peaked as a language model's, and a draft model's that are near them.
    logits = torch.randn((starts[-1], vocab), device=_DEVICE, generator=gen) * 5.0
    target = torch.softmax(logits, dim=-1)
    rows = _ints([starts[b] + i for b, k in enumerate(drafts) for i in range(k)], torch.long)
    probs = None
    if total and case["probs"]:
        probs = torch.softmax(logits[rows] + 0.5 * torch.randn((total, vocab), device=_DEVICE, generator=gen), dim=-1)
    tokens = torch.zeros(0, dtype=torch.long, device=_DEVICE)
    if total:
        # Looked-up drafts are the likely continuation: drawn from a sharpened target.
        source = probs if probs is not None else torch.softmax(3.0 * logits[rows], dim=-1)
        tokens = torch.multinomial(source, 1, generator=gen)[:, 0]
    return {"op": "verify", "target": target, "draft_probs": probs, "drafts": tokens, "query_start": _ints(starts),
            "max_query": max(drafts) + 1, "accept": torch.rand(total, device=_DEVICE, generator=gen),
            "sample": torch.rand(len(drafts), device=_DEVICE, generator=gen)}


# ---------------------------------------------------------------- plain forms
def _rotate(x, cos, sin):
    """x [tokens, heads, d] rotated by [tokens, d] tables, in 32 bits."""

    half = x.shape[-1] // 2
    x, cos, sin = x.float(), cos.float()[:, None], sin.float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:]), dim=-1)


def _round_codes(y, code):
    y = y.clamp(-_TOP[code], _TOP[code])
    return (y.round() if code == "int8" else y).to(_CODE[code])


def _update(codes, scales, new, where, fresh, old, phys, code):
    """Append one side (keys or values) to the touched blocks; returns their values in 32 bits."""

    x = new[where].permute(0, 2, 1, 3)  # [touched, heads, slots, d]
    fresh, old = fresh[:, None, :, None], old[:, None, :, None]
    top = torch.where(fresh, x.abs(), torch.zeros_like(x)).amax(dim=(2, 3))
    before = torch.where(old.any(dim=2)[..., 0], scales[phys], torch.zeros_like(top))
    scale = torch.maximum(before, top / _TOP[code])
    scale = torch.where(scale < _TINY, torch.zeros_like(scale), scale)
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    held = codes[phys].float()
    again = _round_codes(held * (before * inverse)[..., None, None], code).float()
    grown = (scale > before)[..., None, None]
    kept = torch.where(old & grown, again, held)
    coded = torch.where(fresh, _round_codes(x * inverse[..., None, None], code).float(), kept)
    codes[phys] = coded.to(_CODE[code])
    scales[phys] = scale
    return coded * scale[..., None, None]


def _plain_append(s):
    case, act = s["case"], s["qkv"].dtype
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["block"]
    qkv, at = s["qkv"].view(-1, hq + 2 * hkv, d), s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    turned = _rotate(qkv[:, :hq + hkv], cos, sin)
    req, blk = s["touched"]
    computed, start = s["computed"].long()[req][:, None], s["query_start"].long()
    place = blk[:, None] * bs + torch.arange(bs, device=at.device)
    end = computed + (start[req + 1] - start[req])[:, None]
    fresh, old = (place >= computed) & (place < end), place < computed
    where = torch.where(fresh, start[req][:, None] + place - computed, torch.zeros_like(place))
    phys = s["touched_blocks"].long()
    keys = _update(s["keys"], s["key_scales"], turned[:, hq:], where, fresh, old, phys, case["code"])
    values = _update(s["values"], s["value_scales"], qkv[:, hq + hkv:].float(), where, fresh, old, phys, case["code"])
    return {"query": turned[:, :hq].to(act), "keys": keys.to(act), "values": values.to(act)}


def _attend(s, group):
    """Attention of one group of requests, padded to its longest query and context."""

    which, longest, span, rows, slot, place = group
    case = s["case"]
    n, hkv, bs, d = which.shape[0], case["hkv"], case["block"], case["d"]
    heads = case["hq"] // hkv
    table = s["tables"][which][:, :-(-span // bs)].long()

    def read(codes, scales):
        x = codes[table].float() * scales[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)

    keys, values = read(s["keys"], s["key_scales"]), read(s["values"], s["value_scales"])
    q = torch.zeros((n, longest, case["hq"], d), device=keys.device)
    q[slot, place] = s["query"][rows].float()
    q = q.view(n, longest, hkv, heads, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, longest * heads, d)
    score = torch.matmul(q, keys.transpose(2, 3)) * s["scale"]
    last = s["computed"].long()[which][:, None] + torch.arange(longest, device=q.device).repeat_interleave(heads)
    seen = torch.arange(keys.shape[2], device=q.device) <= last[..., None]
    score = score.masked_fill(~seen[:, None], -math.inf)
    score = torch.exp(score - score.amax(dim=-1, keepdim=True))
    out = torch.matmul(score, values) / score.sum(dim=-1, keepdim=True)
    out = out.view(n, hkv, longest, heads, d).permute(0, 2, 1, 3, 4).reshape(n, longest, -1, d)
    return out[slot, place]


def _plain_attention(s):
    out = torch.empty_like(s["query"])
    parts = [(g[3], _attend(s, g)) for g in s["groups"]]
    for rows, values in parts:
        out[rows] = values.to(out.dtype)
    return out


def _plain_verify(s):
    target, drafts, start = s["target"], s["drafts"], s["query_start"].long()
    n, width, vocab = start.shape[0] - 1, s["max_query"], target.shape[1]
    count = start[1:] - start[:-1] - 1
    col = torch.arange(width, device=target.device)
    valid = col < count[:, None]
    first = start[:-1] - torch.arange(n, device=target.device)  # a request's first draft
    accepted = torch.zeros(n, dtype=torch.long, device=target.device)
    grid = torch.full((n, width), -1, dtype=torch.long, device=target.device)
    left = None
    if drafts.shape[0]:
        at = torch.where(valid, first[:, None] + col, torch.zeros_like(valid, dtype=torch.long))
        token = drafts[at]
        p = target[start[:-1, None] + torch.where(valid, col, torch.zeros_like(col)), token]
        q = s["draft_probs"][at, token] if s["draft_probs"] is not None else torch.ones_like(p)
        ok = valid & (s["accept"][at] * q < p)
        accepted = torch.cumprod(ok.long(), dim=1).sum(dim=1)
        grid = torch.where(col < accepted[:, None], token, grid)
        refused = (accepted < count)[:, None]
        row = torch.where(refused[:, 0], first + accepted, torch.zeros_like(first))
        if s["draft_probs"] is not None:
            left = torch.where(refused, s["draft_probs"][row], torch.zeros_like(target[:1]))
        else:
            left = torch.zeros((n, vocab), device=target.device)
            left.scatter_(1, drafts[row][:, None], math.inf)
            left = torch.where(refused, left, torch.zeros_like(left))
    p = target[start[:-1] + accepted]
    rest = p if left is None else p - left

    def fixed(x):
        x = torch.where(x > 0, x, torch.zeros_like(x)).clamp(max=1.0)
        return torch.round(x * 2.0 ** 40).long()

    weight = fixed(rest)
    weight = torch.where(weight.sum(dim=1, keepdim=True) > 0, weight, fixed(p))
    upto = weight.cumsum(dim=1)
    total = upto[:, -1]
    bar = torch.minimum((s["sample"].double() * total.double()).floor().long(), total - 1)
    token = (upto <= bar[:, None]).sum(dim=1).clamp(max=vocab - 1)
    token = torch.where(total > 0, token, torch.full_like(token, vocab - 1))
    grid = torch.where(col == accepted[:, None], token[:, None], grid)
    return {"tokens": grid, "accepted": accepted.to(torch.int32)}


# ------------------------------------------------------- the package's operators
def _own(s):
    from light_vllm_b200 import KV8Layer, KV8Step, kv8_append, kv8_attention, kv8_read_blocks, verify_drafts

    if s["op"] == "verify":
        tokens, accepted = verify_drafts(s["target"], s["drafts"], s["accept"], s["sample"], s["query_start"],
                                         max_query_len=s["max_query"], draft_probs=s["draft_probs"])
        return {"tokens": tokens, "accepted": accepted}
    layer = KV8Layer(s["keys"], s["values"], s["key_scales"], s["value_scales"])
    step = KV8Step(s["tables"], s["computed"], s["query_start"], s["max_query"], s["max_seq"])
    if s["op"] == "attention":
        return kv8_attention(s["query"], layer, step, scale=s["scale"])
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    query, key, value = s["qkv"].view(-1, hq + 2 * hkv, d).split((hq, hkv, hkv), dim=1)
    query = kv8_append(query, key, value, layer, step, positions=s["positions"], cos=s["cos"], sin=s["sin"])
    keys, values = kv8_read_blocks(layer, s["touched_blocks"], dtype=query.dtype)
    return {"query": query, "keys": keys, "values": values}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}[state["op"]](state)


# ------------------------------------------------------------------ what it costs
def work(case):
    if case["op"] == "verify":
        # The probabilities at the drafts, then one target row and, for the about 60 % of requests (model drafts) that
        # have a draft refused, the draft's row.
        drafts = _drafts(case)
        rows = sum(1.0 + (0.6 if k and case["probs"] else 0.0) for k in drafts)
        return {"bytes": rows * case["vocab"] * 4 + sum(drafts) * 24, "flops": rows * case["vocab"] * 2}
    reqs = _requests(case)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["block"]
    tokens = sum(q for _, q in reqs)
    if case["op"] == "append":
        touched = sum(-(-(c + q) // bs) - c // bs for c, q in reqs)
        moved = tokens * (hq + 2 * hkv) * d * 2 + tokens * hq * d * 2 + tokens * d * 2 * 2  # rows, queries, tables
        back = touched * hkv * (bs * d * (1 + 2) + 8) * 2  # the touched blocks: codes read, values written
        return {"bytes": moved + tokens * 2 * hkv * d + back, "flops": tokens * (hq + 2 * hkv) * d * 4}
    pairs = sum(q * c + q * (q + 1) // 2 for c, q in reqs)
    cache = sum(c + q for c, q in reqs) * hkv * 2 * (d + 4 / bs)
    return {"bytes": cache + tokens * hq * d * 2 * 2, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers
    s = prepare(case, seed)
    return (_exact_attention if case["op"] == "attention" else _exact_append)(case, s)


def _exact_attention(case, s):
    hkv, d, bs = case["hkv"], case["d"], case["block"]
    heads = case["hq"] // hkv
    out = torch.empty(s["query"].shape, dtype=torch.float64, device=_DEVICE)
    start = 0
    for r, (computed, queries) in enumerate(_requests(case)):
        span = computed + queries
        blocks = s["tables"][r, : -(-span // bs)].long()
        for h in range(hkv):
            k = s["keys"][blocks, h].float().double() * s["key_scales"][blocks, h].double()[:, None, None]
            v = s["values"][blocks, h].float().double() * s["value_scales"][blocks, h].double()[:, None, None]
            k, v = k.reshape(-1, d)[:span], v.reshape(-1, d)[:span]
            for g in range(heads):
                q = s["query"][start:start + queries, h * heads + g].double()
                score = (q @ k.T) / math.sqrt(d)
                hidden = torch.ones((queries, span), dtype=torch.bool, device=_DEVICE).triu(computed + 1)
                score[hidden] = -math.inf
                out[start:start + queries, h * heads + g] = torch.softmax(score, dim=-1) @ v
        start += queries
    return out


def _exact_append(case, s):
    hq, hkv, d, bs, code = case["hq"], case["hkv"], case["d"], case["block"], case["code"]
    reqs, half = _requests(case), d // 2
    qkv = s["qkv"].view(-1, hq + 2 * hkv, d).double()
    cos, sin = (s[n][s["positions"].long()].double()[:, None, :] for n in ("cos", "sin"))
    flipped = torch.cat((-qkv[..., half:], qkv[..., :half]), dim=-1)
    turned = qkv * cos + flipped * sin
    sides = {"keys": [], "values": []}
    for r, (computed, queries) in enumerate(reqs):
        first = int(s["query_start"][r])
        for b in range(computed // bs, -(-(computed + queries) // bs)):
            low, high = max(computed, b * bs), min(computed + queries, (b + 1) * bs)
            phys, old = int(s["tables"][r, b]), low - b * bs
            rows = slice(first + low - computed, first + high - computed)
            for side, x in (("keys", turned[rows, hq:hq + hkv]), ("values", qkv[rows, hq + hkv:])):
                held = s[side][phys].float().double()
                scale0 = s[side[:-1] + "_scales"][phys].double() if old > 0 else torch.zeros(hkv, dtype=torch.float64, device=_DEVICE)
                scale = torch.maximum(scale0, x.abs().amax(dim=(0, 2)) / _TOP[code])

                def to_code(y):
                    return y.round() if code == "int8" else y.float().to(_CODE[code]).float().double()

                grown = scale > scale0 * (1 + 1e-7)
                ratio = torch.where(grown, scale0 / scale, torch.ones_like(scale))
                held[:, :old] = to_code(held[:, :old] * ratio[:, None, None])
                held[:, old:high - b * bs] = to_code(x.permute(1, 0, 2) / scale[:, None, None])
                sides[side].append(held * scale[:, None, None])
    return {"query": turned[:, :hq], "keys": torch.stack(sides["keys"]), "values": torch.stack(sides["values"])}
