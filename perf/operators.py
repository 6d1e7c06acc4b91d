"""The operators of the 8-bit key/value cache, timed one call at a time.

The cache holds keys and values as e4m3 numbers under a power of two per block of 16 tokens and head:

  append     norm and rotation of a step's queries and keys, and the write of the keys and values into their pages, where a block's
             power grows with what it holds (`ops.qk_norm_rope_store_e4m3`)
  attention  of a step's tokens over the pages, grouped heads, causal, windowed or not (`ops.paged_attention_e4m3`): single tokens
             of decoding requests and portions of prompts

A case names the operator, the heads, a page's tokens and the step: `decode` requests of one token each over up to `context` tokens
(`ragged`: from a twentieth of it on, and every eleventh a padding row that sees nothing), then `prompts` portions of up to `tokens`
tokens behind `before` kept ones. `lengths` seeds the ragged lengths. With `own` the calls are the framework's; else the same is
computed with elementary torch operations in 32 bits. `exact` computes it in 64 bits, request by request.
"""
import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 16                 # tokens under one power of two
LEAST, MOST = -100, 120    # the powers that a block may have
BIAS = 127                 # a block's power is stored with this added, in one byte
TOP = 448.0                # the largest e4m3 number
EPS = 1e-6
SPARE = 5                  # pages that no request holds


def _case(name, op, heads, kv_heads, size, page=16, decode=0, context=0, prompts=0, tokens=0, before=0, ragged=False, window=0, sinks=False, gap=0, lengths=0):
    case = dict(op=op, heads=heads, kv_heads=kv_heads, size=size, page=page, decode=decode, context=context, prompts=prompts, tokens=tokens,
                before=before, ragged=ragged, window=window, sinks=sinks, gap=gap, lengths=lengths)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one user's chat at the smallest Qwen3 sizes: a single new token, where launches and latency count
        _case("append_one", "append", 16, 8, 128, decode=1, context=300),
        # the middle of an offline run: a step of many decoding requests
        _case("append_decode", "append", 16, 8, 128, decode=64, context=2048, ragged=True),
        # a prompt's tokens, from the middle of a block on, out of rows that carry gate columns behind the values
        _case("append_portion", "append", 32, 8, 128, prompts=1, tokens=2048, before=1559, gap=32),
        # a full token budget: ragged prompts beside requests that decode
        _case("append_budget", "append", 32, 8, 128, page=32, decode=60, context=2048, prompts=3, tokens=4096, ragged=True),
        # one user's chat
        _case("decode_one", "attention", 16, 8, 128, decode=1, context=300),
        # the benchmark's default: eight requests of 2,048 tokens
        _case("decode_batch", "attention", 16, 8, 128, decode=8, context=2048),
        # an offline run: many requests of very different lengths, padding rows among them
        _case("decode_ragged", "attention", 32, 8, 128, decode=61, context=4096, ragged=True),
        # long contexts: what the cache is held in 8 bits for
        _case("decode_long", "attention", 32, 8, 128, page=32, decode=8, context=32768),
        # layers with a window and sinks, heads of 64
        _case("window_sinks", "attention", 32, 8, 64, decode=23, context=1700, prompts=2, tokens=1075, ragged=True, window=512, sinks=True),
        # the benchmark's prefill
        _case("prompt", "attention", 16, 8, 128, prompts=1, tokens=2048),
        # serving under a token budget: the next portion of a long prompt
        _case("portion", "attention", 32, 8, 128, page=32, prompts=1, tokens=489, before=7703),
        # a long prompt's first token
        _case("prompt_long", "attention", 32, 8, 128, prompts=1, tokens=8192),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads, size = rng.choice([(16, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128), (32, 8, 64), (16, 4, 64), (16, 2, 256), (6, 2, 32), (8, 8, 80), (12, 1, 48)])
    page, lengths = rng.choice([16, 16, 32, 64, 256]), rng.randrange(1 << 16)
    ragged = rng.random() < 0.6
    if rng.random() < 0.35:
        decode = rng.choice([0, 1, _spread(rng, 1, 128)])
        tokens = _spread(rng, 2, 6000) if not decode or rng.random() < 0.5 else 0
        return _case("", "append", heads, kv_heads, size, page, decode, _spread(rng, 1, 3000) if decode else 0, rng.choice([1, 1, 2]) if tokens else 0, tokens,
                     rng.choice([0, _spread(rng, 1, 3000)]) if tokens else 0, ragged, gap=rng.choice([0, 0, 8, 32]), lengths=lengths)
    window, sinks = rng.choice([0, 0, 0, _spread(rng, 1, 2000)]), rng.random() < 0.3
    kind = rng.choice(["decode", "prompt", "both"])
    decode = _spread(rng, 1, 100) if kind != "prompt" else 0
    context = _spread(rng, 1, min(30000, 260000 // decode)) if decode else 0
    tokens = _spread(rng, 2, 2500) if kind != "decode" else 0
    return _case("", "attention", heads, kv_heads, size, page, decode, context, rng.choice([1, 1, 2, 3]) if tokens else 0, tokens,
                 rng.choice([0, 0, _spread(rng, 1, 4000)]) if tokens else 0, ragged, window, sinks, lengths=lengths)


def _step(case):
    """The step's requests, single tokens first: their new tokens, and their tokens before the step. A padding row has -1 of those."""
    rng = random.Random(case["lengths"])
    some = (lambda n, least: rng.randint(max(least, n // 20), max(least, n))) if case["ragged"] else (lambda n, least: n)
    new, kept = [], []
    for i in range(case["decode"]):
        new.append(1)
        kept.append(-1 if case["ragged"] and i % 11 == 10 else some(case["context"], 1) - 1)
    for _ in range(case["prompts"]):
        new.append(some(case["tokens"], 2))
        kept.append(some(case["before"], 1) if case["before"] else 0)
    return new, kept


def _normal(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _channels(size, gen):
    """Loudness of a head's channels: most alike, a few much louder, as keys have them."""
    loud = torch.rand(size, generator=gen, device=DEV)
    return torch.exp(0.3 * _normal((size,), gen)) * torch.where(loud > 0.96, 6.0, 1.0)


def _filled(shape, blocks_behind, gen, loud):
    """Random numbers under the powers of their blocks: e4m3 bytes of `shape` and the blocks' bytes. `loud` goes by the channel axis."""
    x = _normal(shape, gen).mul_(loud)
    cut = x.unflatten(blocks_behind, (shape[blocks_behind] // BLOCK, BLOCK))
    axes = (3, 4) if blocks_behind == 2 else (2, 4)
    power = torch.ceil(torch.log2(cut.abs().amax(axes, keepdim=True) / TOP)).clamp(LEAST, MOST)
    bits = (cut * torch.exp2(-power)).clamp(-TOP, TOP).to(torch.float8_e4m3fn).flatten(blocks_behind, blocks_behind + 1)
    return bits, (power.squeeze(axes) + BIAS).to(torch.uint8).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    new, kept = _step(case)
    Hq, Hkv, D, page = case["heads"], case["kv_heads"], case["size"], case["page"]
    held = [-(-(n + k) // page) if k >= 0 else 0 for n, k in zip(new, kept)]
    width, pages = max(1, max(held)), sum(held) + SPARE
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, slots, at = [], [], 0
    for n, k, h in zip(new, kept, held):
        mine = order[at:at + h]
        at += h
        tables.append(mine + [-1] * (width - h))
        slots += [mine[p // page] * page + p % page for p in range(k, k + n)] if k >= 0 else [-1] * n
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    loud_k, loud_v = _channels(D, gen), 0.5 + torch.rand(D, generator=gen, device=DEV)
    k, k_scales = _filled((pages, Hkv, page, D), 2, gen, loud_k)
    v, v_scales = _filled((pages, Hkv, D, page), 3, gen, loud_v[:, None])
    T, longest = sum(new), max(n + k for n, k in zip(new, kept))
    state = dict(case=case, k=k, v=v, k_scales=k_scales, v_scales=v_scales)
    if case["op"] == "append":
        angle = torch.arange(max(1, longest), dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
        rows = _normal((T, (Hq + 2 * Hkv) * D + case["gap"]), gen).mul_(torch.exp(0.5 * _normal((T, 1), gen)))
        state |= dict(rows=rows.to(torch.bfloat16)[:, :(Hq + 2 * Hkv) * D], q_weight=1 + 0.2 * _normal((D,), gen), k_weight=loud_k,
                      table=torch.stack((angle.cos(), angle.sin()), -1).float().to(DEV), slots=ints(slots),
                      positions=ints([p for n, k in zip(new, kept) for p in range(max(0, k), max(0, k) + n)]), bound=max(1, longest))
    else:
        cu = [0]
        for n in new[case["decode"]:]:
            cu.append(cu[-1] + n)
        q = _normal((T, Hq * D), gen, torch.bfloat16)
        state |= dict(q=q, tables=ints(tables), contexts=ints([n + k if k >= 0 else 0 for n, k in zip(new, kept)]),
                      positions=ints([p for n, k in zip(new, kept) for p in range(max(0, k), max(0, k) + n)]),
                      seq_of_token=ints([i for i, n in enumerate(new) for _ in range(n)]), cu=ints(cu) if len(cu) > 1 else None,
                      sinks=_normal((Hq,), gen) if case["sinks"] else None, scale=D ** -0.5, most_new=max(new[case["decode"]:], default=0),
                      decode_context=max([n + k for n, k in zip(new, kept)][:case["decode"]], default=0),
                      prefill_context=max([n + k for n, k in zip(new, kept)][case["decode"]:], default=0))
    return state


def run(state):
    if state["case"]["op"] == "append":
        q = _append_own(state) if own else _append_plain(state)
        return {"q": q, "k": state["k"], "v": state["v"], "k_scales": state["k_scales"].view(torch.float8_e8m0fnu),
                "v_scales": state["v_scales"].view(torch.float8_e8m0fnu)}
    return {"o": _attention_own(state) if own else _attention_plain(state)}


# ------------------------------------------------------------------ the framework's calls

def _append_own(s):
    from mini_engine_amd.kernels import ops
    c = s["case"]
    return ops.qk_norm_rope_store_e4m3(s["rows"], s["q_weight"], s["k_weight"], EPS, s["table"], s["positions"], s["slots"],
                                       ops.PagesE4M3(s["k"], s["v"], s["k_scales"], s["v_scales"]), c["heads"], c["kv_heads"], c["size"], c["page"],
                                       position_bound=s["bound"])


def _attention_own(s):
    from mini_engine_amd.kernels import ops
    c = s["case"]
    return ops.paged_attention_e4m3(s["q"], ops.PagesE4M3(s["k"], s["v"], s["k_scales"], s["v_scales"]), c["page"], s["tables"], s["contexts"],
                                    s["seq_of_token"], s["positions"], s["cu"], c["decode"], s["decode_context"], s["scale"], c["window"] or None,
                                    c["heads"], c["kv_heads"], c["size"], max_prefill_context=s["prefill_context"], even_contexts=not c["ragged"],
                                    sinks=s["sinks"])


# ------------------------------------------------------------------ the plain forms

def _normed(x, weight, table, positions):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    turn = table[positions.long()][:, None]
    a, b = x.chunk(2, -1)
    return torch.cat((a * turn[..., 0] - b * turn[..., 1], b * turn[..., 0] + a * turn[..., 1]), -1)


def _place(x, slots, bits, codes, last):
    """x [T, heads, size] into the pages `bits` [pages, heads, page, size] (`last`: [pages, heads, size, page]) and their blocks' bytes
    [pages, heads, blocks of a page], in place. A block's power is the least under which its largest number fits; numbers that were
    there before the first place that is written now keep the block from shrinking, and are rounded again where it grows."""
    pages, heads, per_page = codes.shape
    page, count = per_page * BLOCK, pages * per_page
    spot = torch.where(slots >= 0, slots, count * BLOCK).long()       # rows without a place go to a block that is dropped
    block, place = spot // BLOCK, spot % BLOCK
    largest = x.abs().amax(-1)
    now = torch.zeros(count + 1, heads, device=DEV).scatter_reduce_(0, block[:, None].expand(-1, heads), largest, "amax")[:count]
    first = torch.full((count + 1,), BLOCK, device=DEV).scatter_reduce_(0, block, place, "amin")[:count]
    part, up = torch.frexp(now)
    power = torch.where(now > 0, up - 9 + (part > 0.875), LEAST).clamp(LEAST, MOST)
    old = codes.transpose(1, 2).reshape(count, heads).int() - BIAS
    opened, touched = first == 0, first < BLOCK
    power = torch.where(opened[:, None], power, torch.maximum(power, old))
    power = torch.where(touched[:, None], power, old)
    # [pages, heads, blocks, 16, size]
    held = (bits.transpose(2, 3) if last else bits).float().unflatten(2, (per_page, BLOCK))
    back = torch.exp2((old - power).float()).view(pages, per_page, heads).transpose(1, 2)[..., None, None]
    live = (touched[:, None] & (torch.arange(BLOCK, device=DEV) < first[:, None])).view(pages, 1, per_page, BLOCK, 1)
    held = torch.where(live, held * back, held).to(torch.float8_e4m3fn).flatten(2, 3)
    given = (x * torch.exp2(-power.float())[block.clamp(max=count - 1)][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    # one more page takes the rows without a place
    wide = torch.cat((held.view(torch.uint8), torch.zeros_like(held[:1]).view(torch.uint8)))
    wide[(spot // page)[:, None], torch.arange(heads, device=DEV)[None], (spot % page)[:, None]] = given
    held = wide[:pages]
    bits.view(torch.uint8).copy_(held.transpose(2, 3) if last else held)
    codes.copy_((power + BIAS).view(pages, per_page, heads).transpose(1, 2))


def _append_plain(s):
    c = s["case"]
    Hq, Hkv, D = c["heads"], c["kv_heads"], c["size"]
    rows = s["rows"].unflatten(1, (Hq + 2 * Hkv, D))
    q = _normed(rows[:, :Hq], s["q_weight"], s["table"], s["positions"])
    k = _normed(rows[:, Hq:Hq + Hkv], s["k_weight"], s["table"], s["positions"])
    _place(k, s["slots"], s["k"], s["k_scales"], False)
    _place(rows[:, Hq + Hkv:].float(), s["slots"], s["v"], s["v_scales"], True)
    return q.to(torch.bfloat16).flatten(1)


def _read(bits, codes, tables, last):
    """The requests' keys or values [requests, heads, tokens of the table, size], float32."""
    per_page = codes.shape[2]
    ids = tables.clamp(min=0).long()
    x = bits.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()       # [requests, pages, heads, page, size] (`last`: size, page)
    x = x.transpose(3, 4) if last else x
    scale = torch.exp2(codes[ids].float() - BIAS)                           # [requests, pages, heads, blocks]
    x = x.unflatten(3, (per_page, BLOCK)) * scale[..., None, None]
    return x.flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _softmax_rows(s, q, tables, contexts, counts):
    """q [requests, most new tokens, query heads, size], of which the first counts[r] are there: the last ones of the request."""
    c = s["case"]
    G = c["heads"] // c["kv_heads"]
    k, v = _read(s["k"], s["k_scales"], tables, False), _read(s["v"], s["v_scales"], tables, True)
    B, most = q.shape[:2]
    q = q.float().transpose(1, 2).reshape(B, c["kv_heads"], G * most, c["size"])
    scores = (q @ k.transpose(2, 3).contiguous()).unflatten(2, (G, most)) * s["scale"]
    at = (contexts - counts)[:, None] + torch.arange(most, device=DEV)                     # positions of the rows
    key = torch.arange(k.shape[2], device=DEV)
    seen = (key <= at[..., None]) & (key < contexts[:, None, None])
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    seen = seen[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    sinks = None if s["sinks"] is None else s["sinks"].view(1, c["kv_heads"], G, 1, 1)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = p.flatten(2, 3) @ v
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    o = o.unflatten(2, (G, most)) / torch.where(total > 0, total, 1.0)
    return o.flatten(1, 2).transpose(1, 2)


def _attention_plain(s):
    c = s["case"]
    Hq, D, n = c["heads"], c["size"], c["decode"]
    q, found = s["q"].unflatten(1, (Hq, D)), []
    if n:
        found.append(_softmax_rows(s, q[:n, None], s["tables"][:n], s["contexts"][:n], 1).flatten(0, 1))
    if c["prompts"]:
        cu = s["cu"].long()
        counts = cu[1:] - cu[:-1]
        row = torch.arange(s["most_new"], device=DEV)
        o = _softmax_rows(s, q[n:][(cu[:-1, None] + row).clamp(max=q.shape[0] - n - 1)], s["tables"][n:], s["contexts"][n:], counts)
        request = s["seq_of_token"][n:].long() - n
        found.append(o[request, torch.arange(q.shape[0] - n, device=DEV) - cu[request]])
    return torch.cat(found).to(torch.bfloat16).flatten(1)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    new, kept = _step(case)
    Hq, Hkv, D = case["heads"], case["kv_heads"], case["size"]
    T = sum(new)
    if case["op"] == "append":
        stored = sum(n for n, k in zip(new, kept) if k >= 0)
        # rows, angles, positions and slots in; queries, keys, values and the blocks' bytes out
        return {"bytes": 2 * T * (Hq + 2 * Hkv) * D + 4 * T * D + 8 * T + 2 * T * Hq * D + 2 * stored * Hkv * D + 2 * stored * Hkv // BLOCK,
                "flops": T * D * (10 * (Hq + Hkv) + 4 * Hkv)}
    pairs = read = 0
    for n, k in zip(new, kept):
        if k < 0:
            continue
        sees = lambda at: min(at + 1, case["window"] or at + 1)  # noqa: E731
        pairs += sum(sees(at) for at in range(k, k + n))
        read += min(n + k, (case["window"] or n + k) + n - 1)
    return {"bytes": 4 * T * Hq * D + 2 * read * Hkv * (D + 1 / BLOCK), "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------------ in 64 bits, request by request

def exact(case, seed):
    s = prepare(case, seed)
    return _append_exact(s) if case["op"] == "append" else _attention_exact(s)


def _append_exact(s):
    c = s["case"]
    Hq, Hkv, D, page = c["heads"], c["kv_heads"], c["size"], c["page"]
    x = s["rows"].double().unflatten(1, (Hq + 2 * Hkv, D))
    pos = s["positions"].long()
    cos, sin = (s["table"][pos, :, i].double()[:, None, :] for i in (0, 1))

    def turned(h, w):
        h = h / (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        lo, hi = h[..., :D // 2], h[..., D // 2:]
        return torch.cat((lo * cos - hi * sin, lo * sin + hi * cos), -1)

    k, v = s["k"].double(), s["v"].double()
    kp, vp = (s[n].double() - BIAS for n in ("k_scales", "v_scales"))
    runs, slots = [], s["slots"].tolist()
    for t, slot in enumerate(slots):
        if slot < 0:
            continue
        if runs and runs[-1][1] == t and slots[t - 1] // BLOCK == slot // BLOCK:
            runs[-1][1] = t + 1
        else:
            runs.append([t, t + 1])

    def to_e4m3(y):
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / step) * step

    for new, bits, power, values in ((turned(x[:, Hq:Hq + Hkv], s["k_weight"]), k, kp, False), (x[:, Hq + Hkv:], v, vp, True)):
        for a, b in runs:
            pg, off = slots[a] // page, slots[a] % page
            blk, begin = off // BLOCK, off % BLOCK
            part = bits[pg].transpose(1, 2) if values else bits[pg]                # [heads, page, size], a view
            here = new[a:b].transpose(0, 1)                                         # [heads, run, size]
            need = torch.ceil(torch.log2(here.abs().amax((1, 2)).clamp(min=1e-300) / TOP)).clamp(min=LEAST)
            before = power[pg, :, blk].clone()
            p = torch.maximum(need, before) if begin else need
            if begin:
                live = part[:, off - begin:off]
                part[:, off - begin:off] = to_e4m3(live * torch.exp2(before - p)[:, None, None])
            part[:, off:off + b - a] = to_e4m3(here * torch.exp2(-p)[:, None, None])
            power[pg, :, blk] = p
    return {"q": turned(x[:, :Hq], s["q_weight"]).flatten(1), "k": k, "v": v, "k_scales": torch.exp2(kp), "v_scales": torch.exp2(vp)}


def _attention_exact(s):
    c = s["case"]
    Hq, Hkv, D = c["heads"], c["kv_heads"], c["size"]
    q = s["q"].double().unflatten(1, (Hq, D))
    out = torch.zeros_like(q)
    starts = s["seq_of_token"].tolist()
    for r, L in enumerate(s["contexts"].tolist()):
        rows = [i for i, b in enumerate(starts) if b == r]
        if L == 0:
            continue
        a, n = rows[0], len(rows)
        pages = s["tables"][r, :-(-L // c["page"])].long()
        at = torch.arange(L - n, L, device=DEV)[:, None]
        key = torch.arange(L, device=DEV)[None]
        hidden = key > at
        if c["window"]:
            hidden |= at - key >= c["window"]
        for h in range(Hkv):
            k = s["k"][pages, h].double() * (2.0 ** (s["k_scales"][pages, h].double() - BIAS)).repeat_interleave(BLOCK, 1)[..., None]
            v = s["v"][pages, h].double() * (2.0 ** (s["v_scales"][pages, h].double() - BIAS)).repeat_interleave(BLOCK, 1)[:, None]
            k, v = k.reshape(-1, D)[:L], v.transpose(1, 2).reshape(-1, D)[:L]
            for g in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                z = (q[a:a + n, g] @ k.t()).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
                if s["sinks"] is not None:
                    z = torch.cat((z, s["sinks"][g].double().expand(n, 1)), 1)
                out[a:a + n, g] = torch.softmax(z, -1)[:, :L] @ v
    return {"o": out.flatten(1)}
