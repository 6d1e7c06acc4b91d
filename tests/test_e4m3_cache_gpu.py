"""The 8-bit cache's operators on the GPU against their plain forms in 64 bits."""
import math

import pytest
import torch

from e4m3_cases import (BLOCK, LEAST, PlainPages, Step, attend, attention_bound, empty_pages, mild_pages, normed_rotated, place_bound, power_for,
                        random_pages, rotation)
from mini_engine_amd.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-5


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(T, Hq, Hkv, D, gen, gap=0, offset=0, values_are_keys=False):
    """Packed rows, `gap` columns behind each and `offset` in front of the first: (the view, on the GPU; float64, on the CPU)."""
    width = (Hq + (1 if values_are_keys else 2) * Hkv) * D
    x = torch.randn(T, width, generator=gen) * torch.exp(torch.randn(T, 1, generator=gen))
    flat = torch.zeros(T * (width + gap) + offset, dtype=torch.bfloat16)
    view = flat[offset:].view(T, width + gap)[:, :width]
    view.copy_(x)
    on_gpu = flat.to(DEV)[offset:].view(T, width + gap)[:, :width]
    return on_gpu, view.double()


def _append_plain(rows, step, plain, Hq, Hkv, D, qw, kw, table, values_are_keys=False):
    heads = rows.view(step.T, -1, D)
    q = normed_rotated(heads[:, :Hq], qw, EPS, table, step.positions)
    k = normed_rotated(heads[:, Hq:Hq + Hkv], kw, EPS, table, step.positions)
    v = heads[:, Hq:Hq + Hkv] if values_are_keys else heads[:, Hq + Hkv:]
    plain.place(k, v, step.slots.tolist())
    return q, k, v


def _check_append(rows, q, pages, plain, before, step, exact_k, exact_v, exact_q, values_exact=True):
    T = step.T
    got, stored = PlainPages.of(pages), [t for t in range(T) if step.slots[t] >= 0]
    assert ((q.cpu().double().view(T, -1) - exact_q.reshape(T, -1)).abs() <= (2.0 ** -8 + 2e-6) * exact_q.reshape(T, -1).abs() + 1e-6 * exact_q.abs().max()).all()
    assert torch.equal(got.kp, plain.kp) and torch.equal(got.vp, plain.vp)
    assert torch.equal(got.v, plain.v) or not values_exact
    # keys: half a step of what they round, wherever the rounding falls
    k_now, _ = got.numbers()
    for t in stored:
        pg, off = divmod(int(step.slots[t]), plain.page)
        bound = place_bound(exact_k[t], got.kp[pg, :, off // BLOCK][:, None]) + 1e-6 * exact_k[t].abs().max()
        assert ((k_now[pg, :, off] - exact_k[t]).abs() <= bound).all()
    # places that the call did not write keep their bytes, or are the block's numbers rounded again
    written = torch.zeros(plain.k.shape[0], plain.page, dtype=torch.bool)
    for t in stored:
        written[int(step.slots[t]) // plain.page, int(step.slots[t]) % plain.page] = True
    keep = ~written[:, None, :, None].expand_as(got.k)
    assert torch.equal(got.k[keep], plain.k[keep])


HEADS = [(16, 8, 128), (4, 2, 32), (6, 2, 16), (8, 8, 80), (5, 1, 48), (3, 3, 256), (8, 2, 64), (2, 1, 144)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_append_mixed_step(Hq, Hkv, D, page):
    """Single tokens at every kind of place, a padding row, portions that begin and end inside blocks, out of strided rows."""
    gen = _gen(D + page)
    step = Step([(1, 0), (1, 5), (1, 15), (1, 16), (1, -1), (1, 33), (1, 200), (2, 0), (40, 7), (16, 16), (33, 100)], page, gen)
    pages = random_pages(step.pages, Hkv, D, page, gen)
    plain = PlainPages.of(pages)
    rows, rows64 = _rows(step.T, Hq, Hkv, D, gen, gap=24)
    qw, kw = 1 + 0.2 * torch.randn(D, generator=gen), torch.exp(torch.randn(D, generator=gen))
    table = rotation(256, D)
    kept = rows.clone()
    q = ops.qk_norm_rope_store_e4m3(rows, qw.to(DEV), kw.to(DEV), EPS, table.to(DEV), step.positions.to(DEV), step.slots.to(DEV), pages, Hq, Hkv, D,
                                    page, position_bound=256)
    eq, ek, ev = _append_plain(rows64, step, plain, Hq, Hkv, D, qw, kw, table)
    _check_append(rows, q, pages, plain, None, step, ek, ev, eq)
    assert torch.equal(rows, kept)


@pytest.mark.parametrize("T,before", [(257, 0), (300, 9), (1000, 3), (2049, 0)])
def test_append_long_portion(T, before):
    """More rows than a wave looks at, whole blocks and their ends, beside single tokens."""
    Hq, Hkv, D, page = 4, 2, 64, 32
    gen = _gen(T)
    step = Step([(1, 40), (1, 16), (T, before), (T // 3, 0)], page, gen)
    pages = random_pages(step.pages, Hkv, D, page, gen)
    plain = PlainPages.of(pages)
    rows, rows64 = _rows(step.T, Hq, Hkv, D, gen)
    table = rotation(4096, D)
    w = torch.ones(D)
    q = ops.qk_norm_rope_store_e4m3(rows, w.to(DEV), w.to(DEV), EPS, table.to(DEV), step.positions.to(DEV), step.slots.to(DEV), pages, Hq, Hkv, D, page)
    eq, ek, ev = _append_plain(rows64, step, plain, Hq, Hkv, D, w, w, table)
    _check_append(rows, q, pages, plain, None, step, ek, ev, eq)


@pytest.mark.parametrize("Hkv,D", [(8, 128), (4, 256), (8, 80)])
def test_append_keys_are_the_nearest_numbers(Hkv, D):
    """Of 16 of the power on and up, where a number on the other side of a middle is off by two or more of the power. (In float32 alone one of
    650,000 numbers is on the other side; below, cancellation may leave more than the 2^-20 within which numbers are done again.)"""
    T, page, gen = 3000, 16, _gen(31)
    step = Step([(T, 0), (T, 5000)], page, gen)
    pages = empty_pages(step.pages, Hkv, D, page)
    plain = PlainPages.of(pages)
    rows, rows64 = _rows(step.T, 1, Hkv, D, gen)
    w, table = torch.exp(0.3 * torch.randn(D, generator=gen)), rotation(8192, D)
    ops.qk_norm_rope_store_e4m3(rows, w.to(DEV), w.to(DEV), EPS, table.to(DEV), step.positions.to(DEV), step.slots.to(DEV), pages, 1, Hkv, D, page)
    _append_plain(rows64, step, plain, 1, Hkv, D, w, w, table)
    got = PlainPages.of(pages)
    large = plain.k.abs() >= 16
    assert torch.equal(got.kp, plain.kp) and torch.equal(got.k[large], plain.k[large]) and int(large.sum()) > 0.5 * step.T * Hkv * D


@pytest.mark.parametrize("norm,turn,same", [(False, True, False), (True, False, False), (False, False, False), (True, True, True), (False, False, True)])
@pytest.mark.parametrize("offset", [0, 1])
def test_append_options(norm, turn, same, offset):
    """Without a norm, a rotation, values of their own; rows that begin at an odd address."""
    Hq, Hkv, D, page = 4, 2, 32, 16
    gen = _gen(7)
    step = Step([(1, 3), (1, 0), (20, 13)], page, gen)
    pages = random_pages(step.pages, Hkv, D, page, gen)
    plain = PlainPages.of(pages)
    rows, rows64 = _rows(step.T, Hq, Hkv, D, gen, gap=offset, offset=offset, values_are_keys=same)
    qw, kw = (1 + 0.2 * torch.randn(D, generator=gen), 1 + 0.2 * torch.randn(D, generator=gen)) if norm else (None, None)
    table = rotation(64, D) if turn else None
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    q = ops.qk_norm_rope_store_e4m3(rows, on(qw), on(kw), EPS, on(table), step.positions.to(DEV), step.slots.to(DEV), pages, Hq, Hkv, D, page,
                                    values_are_keys=same)
    eq, ek, ev = _append_plain(rows64, step, plain, Hq, Hkv, D, qw, kw, table, same)
    _check_append(rows, q, pages, plain, None, step, ek, ev, eq)


def test_append_token_by_token():
    """One token after another, growing and not: every step's bytes are the plain form's (no norm, no rotation: nothing is computed)."""
    Hkv, D, page = 3, 48, 16
    gen = _gen(11)
    pages = empty_pages(3, Hkv, D, page)
    plain = PlainPages.of(pages)
    for t in range(40):
        x = torch.randn(1, 2 * Hkv * D, generator=gen) * 10.0 ** float(torch.randint(-3, 4, (1,), generator=gen))
        x = x.to(torch.bfloat16)
        slot = torch.tensor([16 + t if t < 32 else t - 32], dtype=torch.int32)
        ops.qk_norm_rope_store_e4m3(x.to(DEV), None, None, EPS, None, slot.to(DEV), slot.to(DEV), pages, 0, Hkv, D, page)
        h = x.double().view(1, 2 * Hkv, D)
        plain.place(h[:, :Hkv], h[:, Hkv:], [int(slot)])
        got = PlainPages.of(pages)
        assert torch.equal(got.k, plain.k) and torch.equal(got.v, plain.v) and torch.equal(got.kp, plain.kp) and torch.equal(got.vp, plain.vp), t


def test_append_of_nothing_computed_is_the_plain_forms_bytes():
    """Every bfloat16 number of ordinary size, as keys and values; a second identical call changes nothing."""
    Hkv, D, page = 2, 64, 16
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x[torch.isfinite(x.float()) & (x.float().abs() < 3e4)]
    T = x.numel() // (2 * Hkv * D)
    x = x[torch.randperm(x.numel(), generator=_gen(0))][:T * 2 * Hkv * D].view(T, -1)
    pages = empty_pages(-(-T // page) + 1, Hkv, D, page)
    slots = torch.arange(T, dtype=torch.int32) + page
    plain = PlainPages.of(pages)
    h = x.double().view(T, 2 * Hkv, D)
    plain.place(h[:, :Hkv], h[:, Hkv:], slots.tolist())
    for _ in range(2):
        ops.qk_norm_rope_store_e4m3(x.to(DEV), None, None, EPS, None, slots.to(DEV), slots.to(DEV), pages, 0, Hkv, D, page)
        got = PlainPages.of(pages)
        assert torch.equal(got.k, plain.k) and torch.equal(got.v, plain.v) and torch.equal(got.kp, plain.kp) and torch.equal(got.vp, plain.vp)


@pytest.mark.parametrize("slots", [[16] * 40, [16, 17, 18, 17, 18, 19], [20, 19, 18], [3, 3, 3, 0, 1, 1], list(range(16, 32)) * 5 + [16, 17],
                                   [31, 16, 5, -1, 6, -7, 5, 1000, 7], [17] * 100 + [18] * 3, [0] * 300, list(range(16)) * 20])
def test_append_rows_out_of_order(slots):
    """Rows of a block that follow each other out of order are calls one after the other; what a later one opens anew is forgotten.
    Slots that name no place are skipped (1000 lies behind the last page)."""
    Hkv, D, page = 2, 32, 16
    gen = _gen(len(slots))
    pages = random_pages(3, Hkv, D, page, gen)
    plain = PlainPages.of(pages)
    x = (torch.randn(len(slots), 2 * Hkv * D, generator=gen) * torch.exp(2 * torch.randn(len(slots), 1, generator=gen))).to(torch.bfloat16)
    s = torch.tensor(slots, dtype=torch.int32)
    ops.qk_norm_rope_store_e4m3(x.to(DEV), None, None, EPS, None, s.to(DEV), s.to(DEV), pages, 0, Hkv, D, page)
    h = x.double().view(len(slots), 2 * Hkv, D)
    # rows [start, end) of one block; the next ones of the same block that begin at its place 0 make them forgotten
    valid = [v if 0 <= v < 3 * page else -1 for v in slots]
    goes_on = lambda t: t > 0 and valid[t] >= 0 and valid[t - 1] >= 0 and valid[t] // BLOCK == valid[t - 1] // BLOCK  # noqa: E731
    starts = [t for t in range(len(valid)) if not goes_on(t) or valid[t] % BLOCK == 0] + [len(valid)]
    kept = []
    for t, e in zip(starts, starts[1:]):
        if valid[t] >= 0 and not (e < len(valid) and goes_on(e)):
            kept += range(t, e)
    keep = torch.tensor(kept)
    plain.place(h[keep, :Hkv], h[keep, Hkv:], [slots[t] for t in kept])
    got = PlainPages.of(pages)
    # a block whose rows stand apart (others or skipped ones between them) is in no order: any of them may be its last
    apart = [valid[t] // BLOCK for t in range(len(valid)) if valid[t] >= 0 and not goes_on(t)]
    sure = [b for b in range(3) if apart.count(b) <= 1]
    for x, y in ((got.kp, plain.kp), (got.vp, plain.vp), (got.k, plain.k), (got.v, plain.v)):
        assert torch.equal(x[sure], y[sure])


def test_append_numbers_that_are_none():
    """Infinities and NaN are stored as NaN and leave the block's power to the others."""
    Hkv, D, page = 1, 32, 16
    x = torch.randn(4, 2 * D, generator=_gen(1)).to(torch.bfloat16)
    x[0, 3] = math.inf
    x[1, 5] = -math.inf
    x[2, D + 1] = math.nan
    x[3] = math.nan
    pages = empty_pages(2, Hkv, D, page)
    plain = PlainPages.of(pages)
    slots = torch.tensor([16, 17, 18, 0], dtype=torch.int32)
    ops.qk_norm_rope_store_e4m3(x.to(DEV), None, None, EPS, None, slots.to(DEV), slots.to(DEV), pages, 0, Hkv, D, page)
    h = x.double().view(4, 2, D)
    plain.place(h[:, :1], h[:, 1:], slots.tolist())
    got = PlainPages.of(pages)
    assert torch.equal(got.kp, plain.kp) and torch.equal(got.vp, plain.vp) and got.kp[0, 0, 0] == LEAST
    assert torch.equal(torch.isnan(got.k), torch.isnan(plain.k)) and torch.equal(got.k.nan_to_num(), plain.k.nan_to_num())
    assert torch.equal(torch.isnan(got.v), torch.isnan(plain.v)) and torch.equal(got.v.nan_to_num(), plain.v.nan_to_num())


def test_append_no_rows():
    pages = empty_pages(2, 2, 32, 16)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    q = ops.qk_norm_rope_store_e4m3(torch.zeros(0, 8 * 32, dtype=torch.bfloat16, device=DEV), None, None, EPS, None, none, none, pages, 4, 2, 32, 16)
    assert q.shape == (0, 128)


# ------------------------------------------------------------------ attention

def _attention(q, pages, step, scale, Hq, Hkv, D, window=None, chunk=None, sinks=None):
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return ops.paged_attention_e4m3(q, pages, step.page, on(step.tables), on(step.contexts), on(step.seq), on(step.positions), on(step.cu), step.decode,
                                    step.decode_context, scale, window, Hq, Hkv, D, max_prefill_context=step.prefill_context, chunk=chunk, sinks=on(sinks))


def _check_attention(lengths, Hq, Hkv, D, page, seed=0, gap=0, pages=None, loud=1.0, scale=None, **options):
    gen = _gen(seed)
    step = Step(lengths, page, gen)
    pages = mild_pages(step.pages, Hkv, D, page, gen) if pages is None else pages(step, gen)
    q = (loud * torch.randn(step.T, Hq * D + gap, generator=gen)).to(torch.bfloat16)
    scale = D ** -0.5 if scale is None else scale
    got = _attention(q.to(DEV)[:, :Hq * D], pages, step, scale, Hq, Hkv, D, **options)
    o, spread = attend(q[:, :Hq * D].double().view(step.T, Hq, D), PlainPages.of(pages).numbers(), step, scale, Hq, Hkv, **options)
    got = got.cpu().double().view(step.T, Hq, D)
    assert torch.equal(torch.isnan(got), torch.isnan(o))
    off = (got - o).abs() - attention_bound(o, spread)
    assert (off.nan_to_num() <= 0).all(), float(off.nan_to_num().max())
    return got, o, step


MIX = [(1, 0), (1, 1), (1, 62), (1, 63), (1, 64), (1, -1), (1, 300), (1, 255), (2, 0), (65, 0), (7, 130), (129, 16)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS + [(20, 1, 32), (40, 2, 128), (12, 1, 96)])
@pytest.mark.parametrize("page", [16, 128])
def test_attention_mixed_step(Hq, Hkv, D, page):
    """Contexts of one key to several blocks, a padding row, portions of all kinds."""
    _check_attention(MIX, Hq, Hkv, D, page, seed=D, gap=8)


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (6, 2, 32), (5, 1, 48), (8, 8, 80), (8, 2, 64), (40, 2, 128), (3, 3, 256)])
def test_attention_of_portions(Hq, Hkv, D):
    """Tiles that end inside a wave, blocks before, on and behind the diagonal, more than 32 blocks (whose pages are looked up anew)."""
    lengths = [(2, 0), (65, 0), (7, 130), (129, 16), (300, 1500), (257, 31)]
    _check_attention(lengths, Hq, Hkv, D, 16, seed=D)
    _check_attention(lengths, Hq, Hkv, D, 64, seed=D, window=200, sinks=torch.randn(Hq, generator=_gen(1)))


@pytest.mark.parametrize("options", [dict(window=1), dict(window=16), dict(window=63), dict(window=100), dict(chunk=8), dict(chunk=50), dict(window=40, sinks=True),
                                     dict(sinks=True), dict(chunk=64, sinks=True)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 8, 32)])
def test_attention_masks(options, Hq, Hkv, D):
    if options.get("sinks"):
        options = dict(options, sinks=torch.randn(Hq, generator=_gen(5)))
    _check_attention(MIX, Hq, Hkv, D, 16, seed=1, **options)


@pytest.mark.parametrize("lengths", [[(1, 9999)], [(1, 40000), (1, 3)], [(1, 2047)] * 8, [(300, 5000)], [(2, 9000)], [(700, 0), (500, 300)], [(1, 700)] * 70])
@pytest.mark.parametrize("window", [None, 1000])
def test_attention_long(lengths, window):
    """Ranges that are cut into partitions and joined."""
    _check_attention(lengths, 8, 2, 128, 32, seed=2, window=window)


def test_attention_uneven_scores():
    """Loud queries: a few keys have all of the softmax, and the maximum rises again and again."""
    got, o, _ = _check_attention(MIX + [(200, 900)], 4, 2, 64, 16, seed=3, loud=20.0)


@pytest.mark.parametrize("scale", [-0.2, 0.0, float("nan")])
@pytest.mark.parametrize("lengths", [[(1, 40)], [(20, 40)]])
def test_attention_scales_that_are_refused(scale, lengths):
    """As over a cache of the activations' type: scales are positive."""
    with pytest.raises(ops.KernelError, match="scale must be positive"):
        _check_attention(lengths, 4, 2, 64, 16, seed=9, scale=scale)


def test_attention_of_a_small_scale():
    """Every key counts nearly alike."""
    _check_attention(MIX + [(200, 900)], 4, 2, 64, 16, seed=9, scale=1e-3, loud=4.0)


@pytest.mark.parametrize("D", [16, 80, 128, 256])
def test_attention_queries_of_all_sizes(D):
    """Channels of very different sizes, rows of zeros; and a power of two that moves from the scale to the queries changes no bit."""
    gen = _gen(D)
    step = Step(MIX + [(200, 900)], 16, gen)
    pages = mild_pages(step.pages, 2, D, 16, gen)
    q = torch.randn(step.T, 4, D, generator=gen) * torch.exp2(-(torch.arange(D) % 23).float())
    q[::5, 1] = 0.0
    q = q.to(torch.bfloat16).view(step.T, 4 * D)
    got = _attention(q.to(DEV), pages, step, 0.25, 4, 2, D)
    o, spread = attend(q.double().view(step.T, 4, D), PlainPages.of(pages).numbers(), step, 0.25, 4, 2)
    assert ((got.cpu().double().view(step.T, 4, D) - o).abs() <= attention_bound(o, spread)).all()
    for power in (-60, 60):
        moved = _attention((q.float() * 2.0 ** power).to(torch.bfloat16).to(DEV), pages, step, 0.25 * 2.0 ** -power, 4, 2, D)
        assert torch.equal(moved, got)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D", [48, 128])
def test_attention_a_query_that_is_no_number(D, bad):
    """It makes NaN of its row and head and of nothing else."""
    gen = _gen(12)
    step = Step([(1, 300), (1, 700), (40, 0), (130, 400)], 16, gen)
    pages = mild_pages(step.pages, 2, D, 16, gen)
    q = torch.randn(step.T, 4, D, generator=gen).to(torch.bfloat16)
    rows = [1, 41, 42, step.T - 1]
    for r in rows:
        q[r, 2, 5] = bad
    got = torch.isnan(_attention(q.view(step.T, 4 * D).to(DEV), pages, step, 0.2, 4, 2, D).cpu().view(step.T, 4, D))
    assert got[rows, 2].all() and int(got.sum()) == len(rows) * D


@pytest.mark.parametrize("D", [32, 128, 256])
def test_attention_nan_in_a_value(D):
    """A value that is NaN makes NaN of its channel in the rows that see it and of nothing else, on the diagonal, in front of it, under a window
    and where the range is cut into partitions."""
    for new, before, at, window in ((90, 0, 50, None), (70, 700, 720, None), (70, 700, 100, None), (60, 100, 130, 20), (40, 3000, 2999, None)):
        def pages(step, gen):
            p = mild_pages(step.pages, 2, D, 16, gen)
            p.v.view(torch.uint8)[step.table_rows[0][at // 16], 1, 7, at % 16] = 0x7F
            return p
        got, o, step = _check_attention([(new, before)], 4, 2, D, 16, seed=5, pages=pages, window=window)
        seen = sum(1 for i in range(before, before + new) if at <= i and not (window and at <= i - window))
        assert int(torch.isnan(got).sum()) == seen * 2 and torch.isnan(got[:, 2:, 7]).sum() == seen * 2


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (4, 2, 128), (3, 3, 256), (6, 2, 48)])
@pytest.mark.parametrize("new,before,window", [(300, 0, None), (300, 5, 100), (200, 1000, None)])
def test_attention_nan_in_a_later_value(Hq, Hkv, D, new, before, window):
    """A value that is NaN behind a tile's last token changes no bit of the tile's rows, not by another way of computing them either: the walk
    reads up to two blocks further than the rows see."""
    gen, page = _gen(D), 16
    step = Step([(new, before)], page, gen)
    pages = mild_pages(step.pages, Hkv, D, page, gen)
    q = torch.randn(step.T, Hq * D, generator=gen).to(torch.bfloat16).to(DEV)
    clean = _attention(q, pages, step, D ** -0.5, Hq, Hkv, D, window=window)
    tile = 128 // (Hq // Hkv)                 # tokens that lie wholly in the first tile; one more may lie there in part
    for at in (before + -(-128 // (Hq // Hkv)), before + tile + 41):
        one = _copied(pages)
        one.v.view(torch.uint8)[step.table_rows[0][at // page], :, 3, at % page] = 0x7F
        got = _attention(q, one, step, D ** -0.5, Hq, Hkv, D, window=window)
        assert torch.equal(got[:tile], clean[:tile])
        assert torch.isnan(got[at - before].view(Hq, D)[:, 3]).all() and int(torch.isnan(got[at - before]).sum()) == Hq


def test_attention_nan_where_nobody_looks():
    """Foreign and unwritten places hold NaN, in pages of others, behind the context and in front of the window: no row may notice. A key or a
    value that is NaN makes NaN of the rows (the value: of its channel in the rows) that see it, and of no other."""
    def pages(step, gen):
        p = mild_pages(step.pages, 2, 32, 16, gen)
        k, v = p.k.view(torch.uint8), p.v.view(torch.uint8)
        held = {}
        for table, L in zip(step.table_rows, step.contexts.tolist()):
            for i, pg in enumerate(table):
                held[pg] = (i * 16, L)
        for pg in range(step.pages):
            first, L = held.get(pg, (0, 0))
            for off in range(16):
                if first + off >= L or first + off < 3:       # behind the end; in front of what a window of 40 shows the last rows
                    if first + off >= L or L > 60:
                        k[pg, :, off] = 0x7F
                        v[pg, :, :, off] = 0xFF
        return p
    _check_attention([(1, 99), (1, 0), (1, 64), (3, 110), (20, 61)], 4, 2, 32, 16, seed=4, pages=pages, window=40)

    def one_value(step, gen):
        p = mild_pages(step.pages, 2, 32, 16, gen)
        pg = step.table_rows[0][50 // 16]
        p.v.view(torch.uint8)[pg, 1, 7, 50 % 16] = 0x7F
        return p
    got, o, step = _check_attention([(90, 0)], 4, 2, 32, 16, seed=5, pages=one_value)
    assert torch.isnan(got[50:, 2:, 7]).all() and not torch.isnan(got[:50]).any() and int(torch.isnan(got).sum()) == 40 * 2

    def one_key(step, gen):
        p = mild_pages(step.pages, 2, 32, 16, gen)
        p.k.view(torch.uint8)[step.table_rows[0][50 // 16], 1, 50 % 16, 7] = 0xFF
        return p
    gen = _gen(6)
    step = Step([(90, 0)], 16, gen)
    p = one_key(step, gen)
    q = torch.randn(step.T, 128, generator=gen).to(torch.bfloat16).to(DEV)
    got = _attention(q, p, step, 0.2, 4, 2, 32)
    assert torch.isnan(got[50:, 64:].float()).all() and not torch.isnan(got[:50].float()).any() and not torch.isnan(got[:, :64].float()).any()


def test_attention_tables_with_holes():
    """Keys of table entries that hold no page, or name none, are not seen; a row that sees nothing gets zeros."""
    gen = _gen(8)
    step = Step([(1, 100), (1, 20), (30, 40)], 16, gen)
    pages = mild_pages(step.pages, 2, 64, 16, gen)
    for r, i, bad in ((0, 2, -1), (0, 3, 1 << 30), (1, 0, -1), (1, 1, -5), (2, 0, step.pages)):
        step.table_rows[r][i] = -1
        step.tables[r, i] = bad
    q = torch.randn(step.T, 4 * 64, generator=gen).to(torch.bfloat16)
    got = _attention(q.to(DEV), pages, step, 0.1, 4, 2, 64).cpu().double().view(step.T, 4, 64)
    o, spread = attend(q.double().view(step.T, 4, 64), PlainPages.of(pages).numbers(), step, 0.1, 4, 2)
    assert ((got - o).abs() <= attention_bound(o, spread)).all() and not got[1].any()


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (4, 2, 128), (3, 3, 256)])
@pytest.mark.parametrize("hole", [900, 970, 1000, 1030, 1060, 1300])
def test_attention_windows_with_holes(Hq, Hkv, D, hole):
    """A block without a page inside the windows of a tile's first tokens and in front of its last ones', and further on: none of its keys is seen,
    whatever page 0, whose bytes are read in their place, holds."""
    gen, page = _gen(D + hole), 32
    step = Step([(140, 1500)], page, gen)
    pages = mild_pages(step.pages, Hkv, D, page, gen)
    spare = next(p for p in range(step.pages) if p not in step.table_rows[0])
    step.table_rows[0] = [spare if p == 0 else p for p in step.table_rows[0]]
    step.table_rows[0][hole // page] = -1
    step.tables = torch.tensor(step.table_rows, dtype=torch.int32)
    pages.k.view(torch.uint8)[0] = 0x7F
    pages.v.view(torch.uint8)[0] = 0x7F
    q = torch.randn(step.T, Hq * D, generator=gen).to(torch.bfloat16)
    got = _attention(q.to(DEV), pages, step, D ** -0.5, Hq, Hkv, D, window=600).cpu().double().view(step.T, Hq, D)
    numbers = PlainPages.of(pages).numbers()
    for x in numbers:
        x[0] = 0.0            # (the plain form takes its hidden keys from page 0 too, and drops them)
    o, spread = attend(q.double().view(step.T, Hq, D), numbers, step, D ** -0.5, Hq, Hkv, window=600)
    assert ((got - o).abs() <= attention_bound(o, spread)).all()


def test_attention_of_no_rows():
    pages = mild_pages(2, 2, 32, 16, _gen(0))
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    out = ops.paged_attention_e4m3(torch.zeros(0, 128, dtype=torch.bfloat16, device=DEV), pages, 16, torch.zeros(0, 1, dtype=torch.int32, device=DEV), z, z, z,
                                   None, 0, 0, 1.0, None, 4, 2, 32)
    assert out.shape == (0, 128)


def test_the_same_call_gives_the_same_bits():
    gen = _gen(9)
    step = Step([(1, 5000), (1, 100), (300, 2000)], 32, gen)
    pages = mild_pages(step.pages, 2, 128, 32, gen)
    q = torch.randn(step.T, 8 * 128, generator=gen).to(torch.bfloat16).to(DEV)
    first = _attention(q, pages, step, 0.1, 8, 2, 128)
    for _ in range(3):
        assert torch.equal(first, _attention(q, pages, step, 0.1, 8, 2, 128))


def test_a_step_after_another():
    """A prompt in portions and then token by token, appended and attended to through the cache alone: every row against 64 bits."""
    Hq, Hkv, D, page = 8, 2, 64, 16
    gen = _gen(10)
    pages, table = empty_pages(20, Hkv, D, page), rotation(256, D)
    plain = PlainPages.of(pages)
    order = torch.randperm(20, generator=gen).tolist()
    w = torch.ones(D)
    kept = 0
    for n in (50, 1, 1, 37, 1, 70, 1, 1, 1):
        step = Step([(n, kept)], page, gen)
        step.table_rows = [order[:-(-(n + kept) // page)]]
        step.tables = torch.tensor(step.table_rows, dtype=torch.int32)
        step.slots = torch.tensor([order[p // page] * page + p % page for p in range(kept, kept + n)], dtype=torch.int32)
        rows, rows64 = _rows(n, Hq, Hkv, D, gen)
        q = ops.qk_norm_rope_store_e4m3(rows, w.to(DEV), w.to(DEV), EPS, table.to(DEV), step.positions.to(DEV), step.slots.to(DEV), pages, Hq, Hkv, D, page)
        got = _attention(q, pages, step, D ** -0.5, Hq, Hkv, D).cpu().double().view(n, Hq, D)
        eq, ek, ev = _append_plain(rows64, step, plain, Hq, Hkv, D, w, w, table)
        _check_append(rows, q, pages, plain, None, step, ek, ev, eq, values_exact=True)
        o, spread = attend(q.cpu().double().view(n, Hq, D), PlainPages.of(pages).numbers(), step, D ** -0.5, Hq, Hkv)
        assert ((got - o).abs() <= attention_bound(o, spread)).all()
        plain.k = PlainPages.of(pages).k            # the few keys at a rounding's border, as they fell
        kept += n


def test_captured_step_is_replayed():
    """Append and attention in a graph, replayed with other inputs, eager work between the replays; the caches' bytes too."""
    Hq, Hkv, D, page = 8, 2, 128, 16
    gen = _gen(12)
    step = Step([(1, 900), (1, 30), (1, -1), (60, 20)], page, gen)
    pages, other = (mild_pages(step.pages, Hkv, D, page, _gen(13)) for _ in range(2))
    table, w = rotation(1024, D).to(DEV), torch.ones(D, device=DEV)
    rows = torch.zeros(step.T, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=DEV)
    on = {n: getattr(step, n).to(DEV) for n in ("tables", "contexts", "seq", "positions", "cu", "slots")}

    def run(rows, pages):
        q = ops.qk_norm_rope_store_e4m3(rows, w, w, EPS, table, on["positions"], on["slots"], pages, Hq, Hkv, D, page)
        return ops.paged_attention_e4m3(q, pages, page, on["tables"], on["contexts"], on["seq"], on["positions"], on["cu"], step.decode, step.decode_context,
                                        D ** -0.5, None, Hq, Hkv, D, max_prefill_context=step.prefill_context)
    run(rows, pages)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(rows, pages)
    for p, o in zip(pages.tensors(), other.tensors()):
        p.copy_(o) if p.dtype == torch.uint8 else p.view(torch.uint8).copy_(o.view(torch.uint8))
    for seed in range(4):
        x = torch.randn(rows.shape, generator=_gen(seed)).to(torch.bfloat16)
        rows.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(x.to(DEV), other)
        torch.cuda.synchronize()
        live = torch.tensor([i for i in range(step.T) if i != 2], device=DEV)
        assert torch.equal(out[live], eager[live]) and not out[2].any()
        for p, o in zip(pages.tensors(), other.tensors()):
            assert torch.equal(p.view(torch.uint8), o.view(torch.uint8))


def _in_two(rows, pages, step, on, qw, kw, table, Hq, Hkv, D, page, scale, same, **options):
    q = ops.qk_norm_rope_store_e4m3(rows, qw, kw, EPS, table, on["positions"], on["slots"], pages, Hq, Hkv, D, page, values_are_keys=same)
    return ops.paged_attention_e4m3(q, pages, page, on["tables"], on["contexts"], on["seq"], on["positions"], None, step.decode, step.decode_context, scale,
                                    options.get("window"), Hq, Hkv, D, chunk=options.get("chunk"), sinks=options.get("sinks"))


def _copied(pages):
    return ops.PagesE4M3(*(t.clone() for t in pages.tensors()))


def _same_bytes(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.tensors(), b.tensors()))


@pytest.mark.parametrize("Hq,Hkv,D", HEADS + [(32, 2, 64), (15, 1, 112)])
@pytest.mark.parametrize("norm,turn,same,options", [(True, True, False, {}), (False, True, False, dict(window=100)), (True, False, True, dict(sinks=True)),
                                                    (False, False, False, dict(chunk=48)), (True, True, True, dict(window=600, sinks=True))])
def test_decode_step_in_one_launch(Hq, Hkv, D, norm, turn, same, options):
    """The bits and the cache's bytes of the two launches: places of all kinds in a block, blocks that grow, one partition and many, a padding row."""
    gen, page = _gen(D + norm), 32 if same else 16
    step = Step([(1, k) for k in (0, 1, 14, 15, 16, 31, 63, 64, 65, -1, 300, 255, 700, 1029, 5000)], page, gen)
    on = {n: getattr(step, n).to(DEV) for n in ("tables", "contexts", "seq", "positions", "slots")}
    options = dict(options, sinks=torch.randn(Hq, generator=gen).to(DEV)) if options.get("sinks") else options
    rows, _ = _rows(step.T, Hq, Hkv, D, gen, gap=8, values_are_keys=same)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=gen)).to(DEV), torch.exp(torch.randn(D, generator=gen)).to(DEV)) if norm else (None, None)
    table = rotation(8192, D).to(DEV) if turn else None
    one = mild_pages(step.pages, Hkv, D, page, gen)
    two, kept = _copied(one), rows.clone()
    want = _in_two(rows, two, step, on, qw, kw, table, Hq, Hkv, D, page, D ** -0.5, same, **options)
    got = ops.decode_step_attention_e4m3(rows, qw, kw, EPS, table, one, page, on["tables"], on["contexts"], step.decode_context, D ** -0.5,
                                         options.get("window"), Hq, Hkv, D, chunk=options.get("chunk"), sinks=options.get("sinks"), values_are_keys=same)
    assert _same_bytes(one, two) and torch.equal(got, want) and torch.equal(rows, kept) and not got[9].any()


def test_decode_step_rows_that_do_not_fit():
    """Rows off the steps of 16 bytes go to the two launches, which take them, and so do more than 16 query heads to a key head."""
    gen = _gen(3)
    step = Step([(1, 40), (1, 16)], 16, gen)
    pages = mild_pages(step.pages, 2, 32, 16, gen)
    args = (None, None, EPS, None, pages, 16, step.tables.to(DEV), step.contexts.to(DEV), 41, 0.1, None)
    for gap, offset, fits in ((0, 0, True), (8, 8, True), (4, 0, False), (8, 4, False)):
        rows, _ = _rows(2, 4, 2, 32, gen, gap=gap, offset=offset)
        assert ops.decode_step_fuses_e4m3(rows, 4, 2) == fits
        if not fits:
            with pytest.raises(ops.KernelError, match="aligned|alignment"):
                ops.decode_step_attention_e4m3(rows, *args, 4, 2, 32)
    rows, _ = _rows(2, 34, 2, 32, gen)
    assert not ops.decode_step_fuses_e4m3(rows, 34, 2)


def test_decode_steps_one_after_another_in_a_graph():
    """Tokens of several requests one by one across blocks and pages, the step replayed with what a step changes, against the two launches."""
    Hq, Hkv, D, page, B = 8, 4, 128, 16, 5
    gen = _gen(77)
    tables = torch.randperm(B * 8, generator=gen).int().view(B, 8).to(DEV)
    contexts = torch.tensor([1, 16, 40, 63, 64], dtype=torch.int32, device=DEV)
    one = mild_pages(B * 8, Hkv, D, page, gen)
    two, table, w = _copied(one), rotation(256, D).to(DEV), torch.ones(D, device=DEV)
    rows = torch.zeros(B, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=DEV)

    def run():
        return ops.decode_step_attention_e4m3(rows, w, w, EPS, table, one, page, tables, contexts, 128, D ** -0.5, None, Hq, Hkv, D)
    first = _copied(one)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for x, y in zip(one.tensors(), first.tensors()):
        x.view(torch.uint8).copy_(y.view(torch.uint8))
    for i in range(40):
        rows.copy_((1.1 ** i) * torch.randn(rows.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        at = contexts - 1
        slots = tables.gather(1, (at // page).long()[:, None])[:, 0] * page + at % page
        q = ops.qk_norm_rope_store_e4m3(rows, w, w, EPS, table, at, slots.int(), two, Hq, Hkv, D, page)
        want = ops.paged_attention_e4m3(q, two, page, tables, contexts, torch.arange(B, dtype=torch.int32, device=DEV), at, None, B, 128, D ** -0.5, None, Hq, Hkv, D)
        assert torch.equal(out, want) and _same_bytes(one, two)
        contexts += 1


def test_decode_step_without_a_page():
    """A token whose table entry names no page is not written; it sees what the others hold, and nothing of itself."""
    gen = _gen(5)
    step = Step([(1, 40), (1, 16), (1, 0)], 16, gen)
    pages, D = mild_pages(step.pages, 2, 64, 16, gen), 64
    before = _copied(pages)
    tables = step.tables.to(DEV)
    for r, entry in ((0, -1), (1, 1 << 30), (2, -7)):
        tables[r, int(step.contexts[r] - 1) // 16] = entry
    rows = torch.randn(3, 8 * D, generator=gen).to(torch.bfloat16).to(DEV)
    got = ops.decode_step_attention_e4m3(rows, None, None, EPS, None, pages, 16, tables, step.contexts.to(DEV), 41, 0.1, None, 4, 2, D)
    assert _same_bytes(pages, before)
    want = ops.paged_attention_e4m3(rows[:, :4 * D], pages, 16, tables, step.contexts.to(DEV), step.seq.to(DEV), step.positions.to(DEV), None, 3, 41, 0.1, None, 4, 2, D)
    assert torch.equal(got, want) and not got[2].any()
    assert ops.decode_step_attention_e4m3(rows[:0], None, None, EPS, None, pages, 16, tables, step.contexts.to(DEV), 41, 0.1, None, 4, 2, D).shape == (0, 4 * D)


def test_calls_on_two_streams_do_not_meet():
    """Two launches side by side, both cut into partitions, on streams of their own."""
    gen = _gen(14)
    step = Step([(1, 6000), (200, 3000)], 32, gen)
    pages = mild_pages(step.pages, 2, 128, 32, gen)
    qs = [torch.randn(step.T, 8 * 128, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2)]
    expect = [_attention(q, pages, step, 0.1, 8, 2, 128) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    on = {n: getattr(step, n).to(DEV) for n in ("tables", "contexts", "seq", "positions", "cu")}
    torch.cuda.synchronize()
    for _ in range(5):
        found = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                found.append(ops.paged_attention_e4m3(q, pages, 32, on["tables"], on["contexts"], on["seq"], on["positions"], on["cu"], step.decode,
                                                      step.decode_context, 0.1, None, 8, 2, 128, max_prefill_context=step.prefill_context))
        torch.cuda.synchronize()
        for a, b in zip(found, expect):
            assert torch.equal(a, b)


def test_tensors_elsewhere_are_refused():
    gen = _gen(15)
    step = Step([(1, 20)], 16, gen)
    pages = mild_pages(step.pages, 2, 32, 16, gen)
    q = torch.randn(1, 128, generator=gen).to(torch.bfloat16)
    with pytest.raises(ops.KernelError, match="current GPU"):
        _attention(q, pages, step, 0.1, 4, 2, 32)
    with pytest.raises(ops.KernelError, match="current GPU"):
        ops.qk_norm_rope_store_e4m3(torch.zeros(1, 8 * 32, dtype=torch.bfloat16, device=DEV), None, None, EPS, None, step.positions, step.slots.to(DEV), pages, 4,
                                    2, 32, 16)
    with pytest.raises(ops.KernelError, match="beyond the rotation table"):
        ops.qk_norm_rope_store_e4m3(torch.zeros(1, 8 * 32, dtype=torch.bfloat16, device=DEV), None, None, EPS, rotation(8, 32).to(DEV), step.positions.to(DEV),
                                    step.slots.to(DEV), pages, 4, 2, 32, 16, position_bound=21)
