"""The 8-bit cache's operators: what they refuse, and the tests' own plain forms. No GPU."""
import math

import pytest
import torch

from e4m3_cases import LEAST, PlainPages, empty_pages, power_for, to_e4m3
from mini_engine_amd.kernels import build, ops
from mini_engine_amd.kernels.ops import KernelError


def test_rounding_is_the_nearest_number():
    """The plain form's rounding against torch's, for every bfloat16 number up to 448."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    assert torch.equal(to_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("largest,power", [(448.0, 0), (448.0001, 1), (449.0, 1), (896.0, 1), (447.0, 0), (1.75, -8), (1.76, -7), (0.0, LEAST),
                                           (2.0 ** -130, LEAST), (3.3e38, 120), (1.0, -8), (224.0, -1), (224.1, 0)])
def test_power(largest, power):
    assert power_for(largest) == power
    if -100 < power < 120 and largest:
        assert largest <= 448 * 2.0 ** power and largest > 448 * 2.0 ** (power - 1)


def test_plain_pages_keep_what_they_hold():
    """A block that grows keeps its numbers within half a step; one that is opened anew forgets them."""
    p = PlainPages(2, 1, 16, 16)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 1, 16, generator=g, dtype=torch.float64) * torch.tensor([1.0, 10.0, 1000.0]).view(3, 1, 1)
    for t in range(3):
        p.place(x[t:t + 1], x[t:t + 1], [16 + t])
    k, v = p.numbers()
    assert ((k[1, 0, :3] - x[:, 0]).abs() <= 2 ** -3.9 * x[:, 0].abs() + 2.0 ** -9.5 * 2.0 ** p.kp[1, 0, 0]).all()
    assert torch.equal(k[1], v[1])
    p.place(x[:1], x[:1], [16])
    assert p.kp[1, 0, 0] == power_for(float(x[0].abs().max()))


def _append_args(D=32, Hq=4, Hkv=2, page=16, T=3, dtype=torch.bfloat16):
    pages = empty_pages(4, Hkv, D, page, "cpu")
    rows = torch.zeros(T, (Hq + 2 * Hkv) * D, dtype=dtype)
    i32 = torch.zeros(T, dtype=torch.int32)
    return dict(rows=rows, q_weight=torch.ones(D), k_weight=torch.ones(D), eps=1e-6, table=torch.zeros(8, D // 2, 2), positions=i32, slots=i32,
                pages=pages, Hq=Hq, Hkv=Hkv, D=D, page=page)


def _refused(call, args, match, **change):
    with pytest.raises(KernelError, match=match):
        call(**{**args, **change})


def test_append_refusals():
    call = ops.HipBackend().qk_norm_rope_store_e4m3
    a = _append_args()
    P = ops.PagesE4M3
    k, v, ks, vs = a["pages"].tensors()
    _refused(call, a, "bfloat16", rows=a["rows"].float())
    _refused(call, a, "rows must be", rows=a["rows"][:, :-1])
    _refused(call, a, "rows must be", rows=torch.zeros(a["rows"].shape[1], 3, dtype=torch.bfloat16).t())
    _refused(call, a, "rows must be", rows=a["rows"][:1].expand(3, -1))
    _refused(call, a, "rows must be", values_are_keys=True)
    _refused(call, a, "power of two", page=24)
    _refused(call, a, "power of two", page=8)
    _refused(call, a, "pages must be", page=32)
    _refused(call, a, "pages must be", pages=P(k.view(torch.uint8), v, ks, vs))
    _refused(call, a, "pages must be", pages=P(k, k, ks, vs))
    _refused(call, a, "pages must be", pages=P(k[:0], v[:0], ks[:0], vs[:0]))
    _refused(call, a, "pages must be", pages=P(k[:, :1].expand(-1, 2, -1, -1), v, ks, vs))
    _refused(call, a, "powers", pages=P(k, v, ks[:3], vs))
    _refused(call, a, "powers", pages=P(k, v, ks, vs.int()))
    _refused(call, a, "norm weights", q_weight=torch.ones(16))
    _refused(call, a, "norm weights", k_weight=torch.ones(32, dtype=torch.bfloat16))
    _refused(call, a, "both norm weights", k_weight=None)
    _refused(call, a, "rotary table", table=torch.zeros(8, 32, 2))
    _refused(call, a, "rotary table", table=torch.zeros(8, 32))
    _refused(call, a, "int32", positions=a["positions"].long())
    _refused(call, a, "int32", slots=a["slots"][:2])
    _refused(call, a, "head counts", Hkv=0, rows=torch.zeros(3, 128, dtype=torch.bfloat16))
    wide = _append_args(D=272)
    _refused(call, wide, "head size")
    odd = _append_args(D=24)
    _refused(call, odd, "head size")


def _attention_args(D=32, Hq=4, Hkv=2, page=16, decode=2, new=(3,)):
    pages = empty_pages(4, Hkv, D, page, "cpu")
    T, B = decode + sum(new), decode + len(new)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    return dict(q=torch.zeros(T, Hq * D, dtype=torch.bfloat16), pages=pages, page=page, block_tables=torch.zeros(B, 2, dtype=torch.int32),
                context_lens=i32(B), seq_of_token=i32(T), positions=i32(T), prefill_cu=i32(len(new) + 1), num_decodes=decode, max_decode_context=4,
                scale=0.1, window=None, Hq=Hq, Hkv=Hkv, D=D)


def test_attention_refusals():
    call = ops.HipBackend().paged_attention_e4m3
    a = _attention_args()
    _refused(call, a, "bfloat16", q=a["q"].float())
    _refused(call, a, "q must be", q=a["q"][:, :-1])
    _refused(call, a, "q must be", q=a["q"][:1].expand(5, -1))
    _refused(call, a, "block tables", block_tables=a["block_tables"].long())
    _refused(call, a, "block tables", block_tables=a["block_tables"][:2])
    _refused(call, a, "block tables", block_tables=a["block_tables"][:, :0])
    _refused(call, a, "metadata", context_lens=a["context_lens"].long())
    _refused(call, a, "metadata", positions=a["positions"][:2])
    _refused(call, a, "decode count", num_decodes=4)
    _refused(call, a, "decode count", num_decodes=-1)
    _refused(call, a, "exclude", window=3, chunk=4)
    _refused(call, a, "negative", window=-3)
    _refused(call, a, "sinks", sinks=torch.zeros(3))
    _refused(call, a, "sinks", sinks=torch.zeros(4, dtype=torch.bfloat16))
    _refused(call, a, "prefill_cu", prefill_cu=None)
    _refused(call, a, "prefill_cu", prefill_cu=a["prefill_cu"][:1])
    _refused(call, a, "prefill_cu", num_decodes=3)
    _refused(call, a, "power of two", page=8)
    _refused(call, a, "pages must be", Hkv=4)
    _refused(call, a, "no multiple", Hkv=0)
    _refused(call, a, "no multiple", Hkv=8, window=4)
    _refused(call, a, "no multiple", Hkv=3)


def test_decode_step_refusals():
    call = ops.HipBackend().decode_step_attention_e4m3
    D, Hq, Hkv, page, B = 32, 4, 2, 16, 3
    a = dict(rows=torch.zeros(B, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16), q_weight=torch.ones(D), k_weight=torch.ones(D), eps=1e-6,
             table=torch.zeros(8, D // 2, 2), pages=empty_pages(4, Hkv, D, page, "cpu"), page=page, block_tables=torch.zeros(B, 2, dtype=torch.int32),
             context_lens=torch.zeros(B, dtype=torch.int32), max_context=4, scale=0.1, window=None, Hq=Hq, Hkv=Hkv, D=D)
    _refused(call, a, "bfloat16", rows=a["rows"].float())
    _refused(call, a, "rows must be", rows=a["rows"][:, :-1])
    _refused(call, a, "rows must be", values_are_keys=True)
    _refused(call, a, "query heads", Hkv=0)
    _refused(call, a, "query heads", Hkv=3)
    _refused(call, a, "query heads", Hq=34)
    _refused(call, a, "both norm weights", k_weight=None)
    _refused(call, a, "float32", q_weight=torch.ones(D, dtype=torch.bfloat16), k_weight=torch.ones(D, dtype=torch.bfloat16))
    _refused(call, a, "rotary table", table=torch.zeros(8, D, 2))
    _refused(call, a, "beyond the rotation table", max_context=9)
    _refused(call, a, "block tables", block_tables=a["block_tables"][:2])
    _refused(call, a, "block tables", context_lens=a["context_lens"][:2])
    _refused(call, a, "block tables", context_lens=a["context_lens"].long())
    _refused(call, a, "window or a block", window=3, chunk=4)
    _refused(call, a, "window or a block", window=-3)
    _refused(call, a, "sinks", sinks=torch.zeros(3))
    _refused(call, a, "power of two", page=24)
    _refused(call, a, "current GPU" if torch.cuda.is_available() else "GPU")


def test_libraries_of_other_head_sizes_are_refused():
    for D in (0, 8, 24, 272, 512):
        with pytest.raises(build.BuildError, match="multiple of 16"):
            build.attention_e4m3_library(D)


def test_a_call_without_a_gpu_says_so():
    if torch.cuda.is_available():
        pytest.skip("there is a GPU")
    with pytest.raises(KernelError, match="GPU"):
        ops.HipBackend().qk_norm_rope_store_e4m3(**_append_args())
    with pytest.raises(KernelError, match="GPU"):
        ops.HipBackend().paged_attention_e4m3(**_attention_args())


@pytest.mark.parametrize("B,Hq,Hkv,ctx,span", [(1, 16, 8, 1, 0), (1, 16, 8, 300, 0), (8, 32, 8, 32768, 0), (64, 32, 8, 4096, 0), (23, 32, 8, 1700, 512),
                                               (1, 12, 1, 100000, 0), (512, 16, 8, 2048, 0), (1, 16, 2, 1, 7), (3, 64, 1, 1000000, 0), (1, 16, 8, 0, 0)])
def test_partitions_cover_the_keys(B, Hq, Hkv, ctx, span):
    """Every key that a token sees lies in a partition, whatever the position in a block its range begins at."""
    part, parts = ops.decode_partitions_e4m3(B, Hq, Hkv, ctx, span)
    assert parts >= 1 and part % 64 == 0 and part > 0
    worst = min(ctx, span + 63) if span else ctx
    assert part * parts >= worst
    for tokens in (2, 63, 489, 8192):
        part, parts = ops.prompt_partitions_e4m3(tokens, 3, Hq, Hkv, 128, ctx, span)
        assert parts >= 1
        if parts > 1:
            rows = 128 // (Hq // Hkv) + 1         # tokens of a tile at most: its keys begin with its first token's window
            assert part % 64 == 0 and part > 0 and part * parts >= (min(ctx, span + rows + 62) if span else ctx)


@pytest.mark.parametrize("B,Hq,Hkv,D,ctx,span,pieces", [
    (8, 16, 8, 128, 640, 0, 3), (8, 16, 8, 128, 513, 0, 3), (16, 32, 8, 128, 1700, 512, 3), (8, 16, 8, 128, 512, 0, 1), (23, 32, 8, 128, 1700, 512, 1),
    (64, 16, 8, 128, 640, 0, 1), (1, 16, 2, 256, 575, 0, 3), (32, 16, 2, 256, 575, 0, 3), (64, 16, 2, 256, 575, 0, 1), (8, 32, 8, 64, 640, 0, 1),
    (16, 16, 8, 96, 600, 0, 1), (1, 6, 2, 32, 640, 0, 1), (8, 16, 8, 128, 641, 0, 3)])
@pytest.mark.parametrize("even", [False, True])
def test_somewhat_more_than_512_keys_go_by_what_was_timed(B, Hq, Hkv, D, ctx, span, pieces, even):
    part, parts = ops.decode_partitions_e4m3(B, Hq, Hkv, ctx, span, even, D)
    assert parts == pieces and (part == 256 or parts == 1)


def test_nan_is_the_only_number_that_is_not_finite():
    x = torch.tensor([math.inf, -math.inf, math.nan, 1.0], dtype=torch.float64)
    assert torch.isnan(to_e4m3(x)).tolist() == [True, True, True, False]
