"""Plain forms of the 8-bit cache's operators in 64 bits, row by row, and the caches, steps and bounds that their tests use."""
from __future__ import annotations

import math

import torch

from mini_engine_amd.kernels import ops

BLOCK, LEAST, MOST, BIAS = 16, -100, 120, 127


def to_e4m3(x):
    """float64 -> the nearest e4m3 number, ties to even, as float64: 3 digits behind the point from 2^-6 on, steps of 2^-9 below.
    (|x| <= 448, NaN for what is not finite.)"""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, math.nan)


def power_for(largest: float) -> int:
    """The least p with largest <= 448 * 2^p, in [-100, 120]."""
    if largest == 0:
        return LEAST
    part, up = math.frexp(largest)
    return min(MOST, max(LEAST, up - 9 + (part > 0.875)))


class PlainPages:
    """The cache as numbers: what the places hold (units of their block's power) and the powers, float64, on the CPU."""

    def __init__(self, pages: int, Hkv: int, D: int, page: int):
        self.k = torch.zeros(pages, Hkv, page, D, dtype=torch.float64)
        self.v = torch.zeros(pages, Hkv, D, page, dtype=torch.float64)
        self.kp = torch.full((pages, Hkv, page // BLOCK), -BIAS)
        self.vp = self.kp.clone()
        self.page = page

    @classmethod
    def of(cls, pages) -> "PlainPages":
        k = pages.k
        p = cls(k.shape[0], k.shape[1], k.shape[3], k.shape[2])
        p.k, p.v = k.cpu().double(), pages.v.cpu().double()
        p.kp, p.vp = pages.k_scales.cpu().int() - BIAS, pages.v_scales.cpu().int() - BIAS
        return p

    def place(self, k, v, slots):
        """k, v [T, Hkv, D] float64; a run of rows with ascending slots of one block at a time."""
        t, page = 0, self.page
        slots = [int(s) if int(s) < self.k.shape[0] * page else -1 for s in slots]
        while t < len(slots):
            e = t + 1
            if slots[t] < 0:
                t = e
                continue
            while e < len(slots) and slots[e] > slots[e - 1] and slots[e] // BLOCK == slots[t] // BLOCK:
                e += 1
            pg, off = divmod(slots[t], page)
            blk, begin = off // BLOCK, off % BLOCK
            for h in range(k.shape[1]):
                for x, held, power in ((k[t:e, h], self.k[pg, h], self.kp[pg, h]), (v[t:e, h], self.v[pg, h].t(), self.vp[pg, h])):
                    sizes = torch.where(torch.isfinite(x), x.abs(), 0.0)
                    p = power_for(float(sizes.max()))
                    if begin:
                        old = int(power[blk])
                        p = max(p, old)
                        live = held[off - begin:off]
                        live.copy_(to_e4m3(live * 2.0 ** max(old - p, -126)))
                    for i in range(t, e):
                        held[slots[i] % page] = to_e4m3(torch.where(torch.isfinite(x[i - t]), x[i - t], math.nan) * 2.0 ** -p)
                    power[blk] = p
            t = e

    def numbers(self):
        """What the places stand for: k [pages, Hkv, page, D], v [pages, Hkv, page, D]."""
        kp = torch.exp2(self.kp.double()).repeat_interleave(BLOCK, 2)[..., None]
        vp = torch.exp2(self.vp.double()).repeat_interleave(BLOCK, 2)[..., None]
        return self.k * kp, self.v.transpose(2, 3) * vp


def empty_pages(pages: int, Hkv: int, D: int, page: int, device="cuda"):
    z = lambda *s, dt=torch.uint8: torch.zeros(s, dtype=dt, device=device)  # noqa: E731
    return ops.PagesE4M3(z(pages, Hkv, page, D).view(torch.float8_e4m3fn), z(pages, Hkv, D, page).view(torch.float8_e4m3fn),
                         z(pages, Hkv, page // BLOCK), z(pages, Hkv, page // BLOCK))


def random_pages(pages: int, Hkv: int, D: int, page: int, gen, device="cuda"):
    """Random numbers of all sizes, under powers from -12 to 4 (no NaN among them)."""
    def bits(*s):
        b = torch.randint(0, 256, s, generator=gen, dtype=torch.int32)
        return torch.where((b & 0x7F) == 0x7F, b - 40, b).to(torch.uint8).to(device).view(torch.float8_e4m3fn)
    powers = lambda: torch.randint(BIAS - 12, BIAS + 5, (pages, Hkv, page // BLOCK), generator=gen, dtype=torch.int32).to(torch.uint8).to(device)  # noqa: E731
    return ops.PagesE4M3(bits(pages, Hkv, page, D), bits(pages, Hkv, D, page), powers(), powers())


def mild_pages(pages: int, Hkv: int, D: int, page: int, gen, device="cuda"):
    """A cache filled with normally distributed numbers, through the plain form."""
    def half(shape, last):
        x = torch.randn(shape, generator=gen, dtype=torch.float32)
        x = x * torch.exp(0.5 * torch.randn((shape[0], shape[1], 1, 1), generator=gen))
        cut = x.unflatten(3 if last else 2, (page // BLOCK, BLOCK))
        axes = (2, 4) if last else (3, 4)
        p = torch.ceil(torch.log2(cut.abs().amax(axes, keepdim=True) / 448))
        stored = (cut * torch.exp2(-p)).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(shape)
        return stored.to(device), (p.squeeze(axes) + BIAS).to(torch.uint8).contiguous().to(device)
    k, kp = half((pages, Hkv, page, D), False)
    v, vp = half((pages, Hkv, D, page), True)
    return ops.PagesE4M3(k, v, kp, vp)


def normed_rotated(x, weight, eps, table, positions):
    """x [T, H, D] float64."""
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    if table is not None:
        cs = table.double()[positions.long()][:, None]
        a, b = x.chunk(2, -1)
        x = torch.cat((a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]), -1)
    return x


def rotation(positions: int, D: int, theta: float = 1e4):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
    return torch.stack((angle.cos(), angle.sin()), -1).float()


class Step:
    """Requests of one step, single tokens first. lengths: (new tokens, kept tokens) each; kept -1: a padding row."""

    def __init__(self, lengths, page: int, gen, spare: int = 3):
        self.new = [n for n, _ in lengths]
        self.kept = [k for _, k in lengths]
        self.decode = sum(1 for n in self.new if n == 1)
        assert all(n == 1 for n in self.new[:self.decode])
        held = [-(-(n + k) // page) if k >= 0 else 0 for n, k in lengths]
        self.pages, self.page = sum(held) + spare, page
        order = torch.randperm(self.pages, generator=gen).tolist()
        self.table_rows, at = [], 0
        for h in held:
            self.table_rows.append(order[at:at + h])
            at += h
        width = max(1, max(held))
        self.tables = torch.tensor([t + [-1] * (width - len(t)) for t in self.table_rows], dtype=torch.int32)
        self.contexts = torch.tensor([n + k if k >= 0 else 0 for n, k in lengths], dtype=torch.int32)
        pos, slots = [], []
        for (n, k), t in zip(lengths, self.table_rows):
            for p in range(max(k, 0), max(k, 0) + n):
                pos.append(p)
                slots.append(t[p // page] * page + p % page if k >= 0 else -1)
        self.positions, self.slots = torch.tensor(pos, dtype=torch.int32), torch.tensor(slots, dtype=torch.int32)
        self.seq = torch.repeat_interleave(torch.arange(len(self.new)), torch.tensor(self.new)).int()
        cu = [0]
        for n in self.new[self.decode:]:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32) if len(cu) > 1 else None
        self.T = sum(self.new)
        totals = [max(0, n + k) for n, k in lengths]
        self.decode_context, self.prefill_context = max(totals[:self.decode], default=0), max(totals[self.decode:], default=0)


def attend(q, numbers, step: Step, scale, Hq, Hkv, window=None, chunk=None, sinks=None):
    """q [T, Hq, D] float64 on the CPU -> (o, sum_j p_j |v_j| / sum_j p_j), float64 [T, Hq, D]."""
    k_all, v_all = numbers
    o, spread = torch.zeros_like(q), torch.zeros_like(q)
    at = 0
    for n, L, table in zip(step.new, step.contexts.tolist(), step.table_rows):
        rows = slice(at, at + n)
        at += n
        if L == 0:
            continue
        table = torch.tensor(table[:-(-L // step.page)])
        ok = (table >= 0).repeat_interleave(step.page)[:L]
        take = lambda x: x[table.clamp(min=0)].transpose(1, 2).reshape(-1, Hkv, x.shape[-1])[:L]  # noqa: E731
        k, v = take(k_all).repeat_interleave(Hq // Hkv, 1), take(v_all).repeat_interleave(Hq // Hkv, 1)
        i, j = torch.arange(L - n, L)[:, None], torch.arange(L)[None]
        seen = (j <= i) & ok[None]
        if window:
            seen &= j > i - window
        if chunk:
            seen &= j // chunk == i // chunk
        s = torch.einsum("thd,jhd->thj", q[rows], k) * scale
        s = torch.where(seen[:, None], s, -math.inf)
        if sinks is not None:
            s = torch.cat((s, sinks.double().view(1, Hq, 1).expand(n, -1, 1)), 2)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)[..., :L]
        if sinks is not None:
            p = torch.where(seen.any(-1)[:, None, None], p, 0.0)
        # a key that a row does not see has no part in it, whatever its value
        hidden = ~seen[:, None, :, None]
        if not torch.isfinite(v).all():
            vv = torch.where(hidden, 0.0, v.transpose(0, 1)[None])
            o[rows] = (p[..., None] * vv).sum(2)
            spread[rows] = (p[..., None] * vv.abs()).sum(2)
        else:
            o[rows] = torch.einsum("thj,jhd->thd", p, v)
            spread[rows] = torch.einsum("thj,jhd->thd", p, v.abs())
    return o, spread


def attention_bound(o, spread):
    """What the kernels may be off: the result is rounded to bfloat16 (2^-8 of it), and so is every probability before it
    multiplies its value (2^-8 of the values' weighted sizes; where the sum takes the rounded ones too, sum_j p_j e_j (v_j - o) with
    |e_j| <= 2^-8 instead of sum_j p_j e_j v_j: another 2^-8 of the result at most). Sums, scores and exponentials are float32: a score is
    off by about 1e-6 of what its products add up to, some tens, and so is a probability relative to itself, 1e-4 in all."""
    return 2.0 ** -7 * o.abs() + (2.0 ** -8 + 2e-4) * spread + 1e-30


def place_bound(exact, powers):
    """A stored number against what it rounds: half a step, 2^-4 of it or 2^-10 of its power below the normal numbers; 2e-6 of float32 work."""
    return (2.0 ** -4 + 2e-6) * exact.abs() + 2.0 ** -10 * torch.exp2(powers.double()) + 1e-30


# ------------------------------------------------------------------ the engine's bookkeeping without a GPU

def _write_back(plain: PlainPages, pages) -> None:
    pages.k.view(torch.uint8).copy_(plain.k.to(torch.float8_e4m3fn).view(torch.uint8))
    pages.v.view(torch.uint8).copy_(plain.v.to(torch.float8_e4m3fn).view(torch.uint8))
    pages.k_scales.copy_((plain.kp + BIAS).to(torch.uint8))
    pages.v_scales.copy_((plain.vp + BIAS).to(torch.uint8))


class PlainOps:
    """The two operators on tensors anywhere, through the plain forms above; beside `kernel_twins.PlainBackend` for the rest."""

    calls = 0

    @staticmethod
    def qk_norm_rope_store_e4m3(rows, q_weight, k_weight, eps, table, positions, slots, pages, Hq, Hkv, D, page, position_bound=0, values_are_keys=False):
        PlainOps.calls += 1
        assert table is None or position_bound <= table.shape[0]
        assert pages.check("append", Hkv, D, page) == pages.k.shape[0]
        on = lambda t: None if t is None else t.cpu()  # noqa: E731
        heads = rows.cpu().double().view(rows.shape[0], -1, D)
        q = normed_rotated(heads[:, :Hq], on(q_weight), eps, on(table), positions.cpu())
        k = normed_rotated(heads[:, Hq:Hq + Hkv], on(k_weight), eps, on(table), positions.cpu())
        plain = PlainPages.of(pages)
        plain.place(k, heads[:, Hq:Hq + Hkv] if values_are_keys else heads[:, Hq + Hkv:], slots.tolist())
        _write_back(plain, pages)
        return q.reshape(rows.shape[0], Hq * D).to(rows)

    @staticmethod
    def paged_attention_e4m3(q, pages, page, block_tables, context_lens, seq_of_token, positions, prefill_cu, num_decodes, max_decode_context, scale,
                             window, Hq, Hkv, D, max_prefill_context=0, even_contexts=False, chunk=None, sinks=None):
        contexts = context_lens.tolist()
        cu = list(range(num_decodes)) + [num_decodes + c for c in (prefill_cu.tolist() if prefill_cu is not None else [0])]
        new = [b - a for a, b in zip(cu, cu[1:])]
        assert max(contexts[:num_decodes], default=0) <= max_decode_context and max(contexts[num_decodes:], default=0) <= max_prefill_context
        step = Step.__new__(Step)
        step.new, step.page, step.contexts = new, page, torch.tensor(contexts)
        step.table_rows = [[int(p) if 0 <= p < pages.k.shape[0] else -1 for p in row] for row in block_tables.tolist()]
        o, _ = attend(q.cpu().double().view(q.shape[0], Hq, D), PlainPages.of(pages).numbers(), step, scale, Hq, Hkv, window, chunk,
                      None if sinks is None else sinks.cpu())
        return o.reshape(q.shape).to(q)
