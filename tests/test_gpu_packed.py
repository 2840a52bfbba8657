"""The operators on packed documents (axis positions, rotation over several
axes, masked attention) against plain 64-bit forms, at the sizes, masks,
strides and types where they can go wrong. packed_ref derives the tolerances."""
import concurrent.futures
import math

import numpy as np
import pytest
import torch

import packed_ref as R
import svl_amd
import svl_packed as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def normal(rng, shape, dtype, gain=1.0):
    """A tensor and its values in 64 bits."""
    t = torch.from_numpy((rng.standard_normal(shape) * gain).astype(np.float32)).to(dtype)
    return t.to(DEV), t.double().numpy()


def host(t):
    return t.double().cpu().numpy()


def within(got, want, bound, what=""):
    assert np.isfinite(got).all(), what
    over = np.abs(got - want) - bound
    assert (over <= 0).all(), f"{what}: {np.abs(got - want).max():.3g} off, {over.max():.3g} too far"


# ---- positions ---------------------------------------------------------------------

def run_positions(segments):
    plan = P.PositionPlan(segments)
    out = torch.full((plan.tokens, 3), -7, dtype=torch.int32, device=DEV)
    P.axis_positions(plan, out)
    return out.cpu().numpy()


@pytest.mark.parametrize("segments", [
    [], [(0, 0, 1, 0, 0, 0)], [(5, 1, 1, 1, 1, 1)], [(0, 0, 0, 0, 0, 0), (0, 1, 3, 0, 4, 1)],
    [(0, 0, 5, 0, 0, 0), (0, 1, 4, 3, 7, 2), (0, 0, 2, 0, 0, 0), (1, 0, 3, 0, 0, 0),
     (1, 1, 1, 9, 2, 1), (1, 1, 0, 3, 3, 1), (1, 0, 6, 0, 0, 0), (7, 1, 5, 1, 1, 100)],
    [(d, 0, 1, 0, 0, 0) for d in range(3000)],                 # a segment for every token
    [(d // 3, d % 2, 1 + d % 5, 1 + d % 7, 1 + d % 4, 1 + d % 3) for d in range(900)],
    [(0, 1, 3, 40, 50, 3), (0, 0, 1023, 0, 0, 0), (0, 0, 1, 0, 0, 0), (2, 1, 1, 32, 32, 1)]])
def test_positions(segments):
    np.testing.assert_array_equal(run_positions(segments), R.positions(segments))


def test_positions_into_rows_off_sixteen_bytes():
    seg = [(0, 0, 9, 0, 0, 0), (0, 1, 2, 5, 3, 1)]
    plan = P.PositionPlan(seg)
    flat = torch.full((3 * plan.tokens + 2,), -7, dtype=torch.int32, device=DEV)
    P.axis_positions(plan, flat[1:-1].view(-1, 3))
    got = flat.cpu().numpy()
    np.testing.assert_array_equal(got[1:-1].reshape(-1, 3), R.positions(seg))
    assert got[0] == got[-1] == -7


def test_positions_refuse_other_tensors():
    plan = P.PositionPlan([(0, 0, 4, 0, 0, 0)])
    for out in (torch.empty(3, 3, dtype=torch.int32, device=DEV),
                torch.empty(4, 3, dtype=torch.int64, device=DEV),
                torch.empty(4, 6, dtype=torch.int32, device=DEV)[:, ::2],
                torch.empty(4, 3, dtype=torch.int32)):
        with pytest.raises(svl_amd.SvlError) as e:
            P.axis_positions(plan, out)
        assert e.value.kind == "Usage"


# ---- rotation ----------------------------------------------------------------------

def axes_of(pairs, order):
    if order == "runs":
        return np.array([0] * (pairs - 2 * (pairs // 3)) + [1] * (pairs // 3) + [2] * (pairs // 3),
                        np.uint8)
    return np.arange(pairs).astype(np.uint8) % 3     # interleaved


def freqs(pairs):
    return (10000.0 ** (-np.arange(pairs) / max(pairs, 1))).astype(np.float32)


def check_rope(rng, tokens, heads, kv, hd, pairs, layout, order, dtype, far=0, inplace=False,
               arrange=lambda x: x):
    axis, freq = axes_of(pairs, order), freqs(pairs)
    pos = rng.integers(-50, 3000, (tokens, 3)).astype(np.int32) + np.int32(far)
    q, q64 = normal(rng, (tokens, heads, hd), dtype)
    k, k64 = normal(rng, (tokens, kv, hd), dtype) if kv else (None, None)
    q, k = arrange(q), None if k is None else arrange(k)
    oq = q if inplace else arrange(torch.full_like(q, 9.0))
    ok = None if k is None else (k if inplace else arrange(torch.full_like(k, 9.0)))
    P.rope_axes(q, k, torch.from_numpy(pos).to(DEV), freq, axis, layout, oq, ok)
    for x, y in ((q64, oq), (k64, ok)):
        if y is None:
            continue
        want = R.rope(x, pos, freq, axis, layout)
        within(host(y), want, R.rope_bound(x, want, axis, layout, dtype == BF16))
        np.testing.assert_array_equal(host(y)[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout,order", [("half", "runs"), ("half", "mixed"), ("adjacent", "mixed"),
                                          ("axial", "runs")])
@pytest.mark.parametrize("tokens,heads,kv,hd,pairs", [
    (1, 1, 1, 2, 1), (5, 3, 1, 256, 128), (301, 12, 12, 64, 30), (64, 4, 2, 128, 32),
    (3, 2, 0, 37, 18), (130, 1, 1, 48, 24), (2, 5, 5, 512, 256), (9, 2, 2, 26, 9),
    (4, 3, 1, 64, 0), (700, 1, 0, 64, 30), (1000, 1, 0, 8, 3), (3, 1, 1, 1024, 255)])
def test_rotation(tokens, heads, kv, hd, pairs, layout, order, dtype):
    check_rope(np.random.default_rng(tokens + hd), tokens, heads, kv, hd, pairs, layout, order,
               dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["half", "adjacent", "axial"])
@pytest.mark.parametrize("hd,pairs", [(64, 24), (64, 30), (37, 7), (256, 128)])
def test_rotation_in_place(hd, pairs, layout, dtype):
    check_rope(np.random.default_rng(4), 77, 3, 1, hd, pairs, layout, "runs", dtype, inplace=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,hd,pairs", [(64, 8, 256, 120), (40, 40, 128, 64), (3, 3, 1024, 250),
                                               (70, 0, 33, 16)])
def test_rotation_of_many_heads(heads, kv, hd, pairs, dtype):
    """More values a token than a workgroup's threads hold at once."""
    for layout in ("half", "axial"):
        check_rope(np.random.default_rng(7), 9, heads, kv, hd, pairs, layout, "runs", dtype)


@pytest.mark.parametrize("far", [10**6, 2**31 - 4000, -2**31 + 100])
def test_rotation_far_out(far):
    check_rope(np.random.default_rng(5), 40, 2, 1, 128, 64, "half", "mixed", F32, far=far)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("arrange", [
    lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),                    # head-major
    lambda x: torch.cat([x, x, x], 1)[:, x.shape[1]:2 * x.shape[1]],             # a fused row's part
    lambda x: torch.cat([x[..., :1], x, x[..., :2]], 2)[..., 1:-2],              # off alignment
    lambda x: torch.cat([x, x], 0).view(2, *x.shape).transpose(0, 1).reshape(-1, *x.shape[1:])[::2]])
def test_rotation_strides(arrange, dtype):
    check_rope(np.random.default_rng(6), 33, 4, 2, 64, 32, "half", "runs", dtype,
               arrange=arrange)


def test_rotation_passes_non_finite_values():
    x = torch.ones(2, 1, 4, device=DEV)
    x[0, 0, 1] = math.inf
    x[1, 0, 0] = math.nan
    y = torch.empty_like(x)
    P.rope_axes(x, None, torch.zeros(2, 1, dtype=torch.int32, device=DEV), np.ones(1, np.float32),
                np.zeros(1, np.uint8), "half", y, None)
    assert not torch.isfinite(y[0, 0, :2]).all() and torch.isnan(y[1, 0, 0])
    assert (y[:, :, 2:] == 1).all()


def test_rotation_refuses_other_tensors():
    q = torch.zeros(4, 2, 8, device=DEV)
    pos = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    f, a = np.ones(4, np.float32), np.zeros(4, np.uint8)
    bad = [(q, None, pos.long(), f, a, "half", q, None), (q, None, pos[:3], f, a, "half", q, None),
           (q, None, pos, f, a[:3], "half", q, None), (q, None, pos, f, a, "whole", q, None),
           (q, q, pos, f, a, "half", q, None), (q, q.bfloat16(), pos, f, a, "half", q, q.bfloat16()),
           (q[0], None, pos, f, a, "half", q[0], None), (q, None, pos, f, a, "half", q[:, :1], None),
           (q, None, pos.cpu(), f, a, "half", q, None), (q, None, pos, f, a + 2, "half", q, None),
           (q.transpose(1, 2), None, pos, f[:1], a[:1], "half", q.transpose(1, 2), None)]
    for args in bad:
        with pytest.raises(svl_amd.SvlError) as e:
            P.rope_axes(*args)
        assert e.value.kind == "Usage"
    with pytest.raises(svl_amd.SvlError) as e:
        P.rope_axes(q.half(), None, pos, f, a, "half", q.half(), None)
    assert e.value.kind == "Unsupported"


# ---- attention ---------------------------------------------------------------------

def offsets(lengths, start=0):
    return np.concatenate([[start], start + np.cumsum(lengths)]).astype(np.int64)


def check_attention(seed, ql, kl, nh, nkv, hd, dtype, *, causal=False, window=None, prefix=None,
                    cap=0.0, slopes=False, scale=None, gain=1.5, start=0, after=0,
                    arrange=lambda x: x, poison=False):
    rng = np.random.default_rng(seed)
    qo, ko = offsets(ql, start), offsets(kl, start)
    q, q64 = normal(rng, (int(qo[-1]) + after, nh, hd), dtype, gain)
    k, k64 = normal(rng, (int(ko[-1]) + after, nkv, hd), dtype)
    v, v64 = normal(rng, (int(ko[-1]) + after, nkv, hd), dtype)
    if poison:   # keys that no query may see
        seen = np.zeros(k.shape[0], bool)
        for d in range(len(ql)):
            if ql[d]:
                m, _ = R.visible(ql[d], kl[d], causal, window, prefix[d] if prefix else 0)
                seen[ko[d]:ko[d + 1]] = m.any(0)
        hidden = torch.from_numpy(~seen).to(DEV)
        k[hidden] = math.nan
        v[hidden] = math.inf
    scale = 1 / math.sqrt(hd) if scale is None else scale
    slope = np.array([2.0 ** (-8 * (h + 1) / nh) for h in range(nh)], np.float32) if slopes else None
    plan = P.AttentionPlan(qo, ko, num_heads=nh, num_kv_heads=nkv, head_dim=hd, dtype=dtype,
                           causal=causal, window=window, prefix=prefix)
    q, k, v = arrange(q), arrange(k), arrange(v)
    out = arrange(torch.full(q.shape, 5.0, dtype=dtype, device=DEV))
    lse = torch.full(q.shape[:2], 5.0, dtype=F32, device=DEV)
    P.masked_attention(plan, q, k, v, out, scale, soft_cap=cap, lse=lse,
                       slopes=None if slope is None else torch.from_numpy(slope).to(DEV))
    want, wlse, ob, lb = R.attention(q64, k64, v64, qo, ko, causal=causal, window=window,
                                     prefix=prefix, scale=scale, cap=cap, slopes=slope,
                                     bf16=dtype == BF16)
    got, glse = host(out), host(lse)
    live = ~np.isnan(wlse)
    assert (got[~live] == 5).all() and (glse[~live] == 5).all()
    within(got[live], want[live], ob[live], "out")
    none = live & (wlse == -np.inf)
    assert (glse[none] == -np.inf).all() and (got[none] == 0).all()
    some = live & ~none
    within(glse[some], wlse[some], lb[some], "lse")
    return plan


TYPES = [F32, BF16]
HEADS = [(3, 1, 256), (12, 12, 64), (4, 2, 128), (4, 1, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS + [(2, 2, 8), (3, 3, 80), (2, 1, 96), (6, 2, 33),
                                               (1, 1, 1), (2, 1, 200), (2, 1, 300), (4, 1, 512),
                                               (1, 1, 1024), (10, 2, 40)])
def test_attention_head_layouts(nh, nkv, hd, dtype):
    check_attention(hd, [1, 65, 130], [1, 65, 130], nh, nkv, hd, dtype)


MASKS = [dict(), dict(causal=True), dict(window=0), dict(window=20), dict(causal=True, window=33),
         dict(causal=True, prefix=[0, 1, 70, 500]), dict(window=5, prefix=[3, 0, 64, 65]),
         dict(causal=True, window=1, prefix=[9, 128, 0, 2])]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_masks(nh, nkv, hd, mask, dtype):
    kl = [300, 1, 129, 64]
    check_attention(1, kl, kl, nh, nkv, hd, dtype, **mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_single_queries(nh, nkv, hd, mask, dtype):
    """One query a document, some over keys enough for several tile ranges, one over none."""
    check_attention(2, [1, 1, 1, 1], [2500, 1, 0, 777], nh, nkv, hd, dtype, **mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", MASKS)
def test_attention_later_part_of_a_prompt(mask, dtype):
    """Queries that begin inside their keys, documents without queries, more queries than keys
    (whose first rows see nothing under a causal mask)."""
    check_attention(3, [40, 0, 150, 90], [400, 50, 151, 20], 4, 2, 128, dtype, **mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("extra", [dict(cap=50.0, gain=8.0), dict(cap=5.0, gain=8.0),
                                   dict(slopes=True), dict(cap=20.0, slopes=True, causal=True),
                                   dict(scale=-0.1), dict(scale=0.0), dict(cap=0.01), dict(cap=1e-39),
                                   dict(cap=1e4, gain=20.0)])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_cap_and_bias(nh, nkv, hd, extra, dtype):
    check_attention(4, [200, 1, 77], [200, 900, 130], nh, nkv, hd, dtype, **extra)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(1, 1, 64), (5, 1, 64), (8, 1, 128), (1, 1, 128), (1, 1, 256),
                                       (9, 1, 128), (40, 1, 64), (6, 3, 100), (3, 1, 250),
                                       (8, 1, 256), (2, 1, 512), (4, 1, 500), (33, 1, 512)])
def test_attention_single_queries_by_their_count(nh, nkv, hd, dtype):
    """One query of one to forty heads a KV head, over keys split many and few ways."""
    check_attention(15, [1, 1, 1], [9000, 3, 400], nh, nkv, hd, dtype, causal=True, slopes=nh > 4,
                    cap=30.0 if hd == 128 else 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 128), (3, 1, 256), (2, 2, 64), (2, 1, 100), (4, 1, 512),
                                       (2, 1, 300)])
def test_attention_few_long_prompts(nh, nkv, hd, dtype):
    """Few groups of many queries, whose keys are split."""
    check_attention(16, [70, 33], [3500, 2000], nh, nkv, hd, dtype, causal=True,
                    prefix=[100, 0], window=None if hd == 64 else 1500)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[], [0], [0, 0, 3], [5] * 200, [1000], [127, 128, 129],
                                     [31, 32, 33, 63, 64, 65]])
def test_attention_lengths(lengths, dtype):
    check_attention(5, lengths, lengths, 4, 2, 64, dtype, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_many_documents_and_heads(dtype):
    check_attention(20, [1] * 3000, [1 + i % 7 for i in range(3000)], 2, 1, 16, dtype)
    check_attention(21, [1, 2], [300, 70], 128, 1, 64, dtype, causal=True)
    check_attention(22, [3], [90], 130, 65, 40, dtype, slopes=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_leaves_rows_outside_documents(dtype):
    check_attention(6, [70, 9], [70, 9], 2, 1, 64, dtype, start=3, after=40, poison=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ql,mask", [([1, 1], dict(window=30)), ([1, 1], dict(causal=True, window=9, prefix=[5, 200])),
                                     ([20, 300], dict(causal=True, window=50)),
                                     ([33, 1], dict(window=0, prefix=[2, 0])),
                                     ([0, 140], dict(causal=True))])
def test_attention_reads_nothing_hidden_from_all(ql, mask, dtype):
    """Keys hidden from every query hold NaN, their values infinities."""
    check_attention(7, ql, [260, 700], 4, 2, 128, dtype, poison=True, **mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS + [(2, 1, 72), (2, 1, 300), (1, 1, 700)])
def test_attention_values_hidden_from_some(nh, nkv, hd, dtype):
    """Under a causal mask a row's own non-finite value reaches it and those after it, and no
    other."""
    rng = np.random.default_rng(8)
    n, bad = 200, 90
    plan = P.AttentionPlan([0, n], num_heads=nh, num_kv_heads=nkv, head_dim=hd, dtype=dtype,
                           causal=True)
    (q, q64), (k, k64), (v, v64) = (normal(rng, (n, h, hd), dtype) for h in (nh, nkv, nkv))
    out = torch.empty_like(q)
    # rows before see neither, and may be summed another way beside such values: the bound of the
    # 64-bit form holds for them either way
    want, _, bound, _ = R.attention(q64, k64, v64, [0, n], [0, n], causal=True, scale=0.1,
                                    bf16=dtype == BF16)
    for key, value in ((math.nan, math.nan), (1.0, math.inf), (math.inf, -math.inf)):
        kk, vv = k.clone(), v.clone()
        kk[bad], vv[bad] = key, value
        P.masked_attention(plan, q, kk, vv, out, 0.1)
        within(host(out[:bad]), want[:bad], bound[:bad])
        assert not torch.isfinite(out[bad]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("arrange", [
    lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
    lambda x: torch.cat([x, x, x], 1)[:, x.shape[1]:2 * x.shape[1]],
    lambda x: torch.cat([x[..., :1], x, x[..., :2]], 2)[..., 1:-2],
    lambda x: torch.stack([x, x], 1)[:, 0]])
def test_attention_strides(arrange, dtype):
    check_attention(9, [90, 40], [90, 40], 4, 2, 64, dtype, arrange=arrange, causal=True)


@pytest.mark.parametrize("dtype,queries", [(BF16, 1), (BF16, 40), (F32, 1), (F32, 40)])
def test_attention_of_a_cache_past_32_bits(dtype, queries):
    """Two documents of 4.5 million keys, 2.3 * 10^9 values, seen through a window at their ends:
    equal to the plain form on those keys alone."""
    hd, each, window = 256, 4_500_000, 150
    g = torch.Generator(device=DEV).manual_seed(3)
    k = torch.empty(2 * each, 1, hd, dtype=dtype, device=DEV).normal_(generator=g)
    v = torch.empty(2 * each, 1, hd, dtype=dtype, device=DEV).normal_(generator=g)
    q = torch.empty(2 * queries, 3, hd, dtype=dtype, device=DEV).normal_(generator=g)
    assert k.numel() > 2**31
    plan = P.AttentionPlan([0, queries, 2 * queries], [0, each, 2 * each], num_heads=3, num_kv_heads=1,
                           head_dim=hd, dtype=dtype, causal=True, window=window)
    assert plan.workspace_bytes < 2**22
    out = torch.empty_like(q)
    P.masked_attention(plan, q, k, v, out, 1 / 16)
    n = queries + window     # the last queries' keys
    last = torch.cat([torch.arange(e - n, e) for e in (each, 2 * each)])
    want, _, bound, _ = R.attention(host(q), host(k[last]), host(v[last]),
                                    [0, queries, 2 * queries], [0, n, 2 * n], causal=True,
                                    window=window, scale=1 / 16, bf16=dtype == BF16)
    within(host(out), want, bound)


def test_attention_keys_of_one_row():
    """Expanded keys: a token stride of 0."""
    rng = np.random.default_rng(10)
    q, q64 = normal(rng, (50, 2, 64), F32)
    k, k64 = normal(rng, (1, 1, 64), F32)
    v, v64 = normal(rng, (50, 1, 64), F32)
    out = torch.empty_like(q)
    plan = P.AttentionPlan([0, 50], num_heads=2, num_kv_heads=1, head_dim=64, dtype=F32)
    P.masked_attention(plan, q, k.expand(50, 1, 64), v, out, 0.125)
    want, _, bound, _ = R.attention(q64, np.repeat(k64, 50, 0), v64, [0, 50], [0, 50], scale=0.125)
    within(host(out), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scores_past_the_range_of_exponentials(dtype):
    """Scores of +-10^5: one key takes all the weight, v p / p. p need not be one (a kernel may keep
    a maximum some powers of two behind), so the result is not v to the bit: in 32 bits the product of three
    parts by three rounds at each of its six sums and leaves out 2 half steps, 1 / p is off by up
    to 2 and the last product by one, 12 in all; in bfloat16 p and the result are rounded to it."""
    rng = np.random.default_rng(11)
    q, q64 = normal(rng, (70, 2, 64), dtype, 300.0)
    k, k64 = normal(rng, (70, 2, 64), dtype, 300.0)
    v, v64 = normal(rng, (70, 2, 64), dtype)
    out = torch.empty_like(q)
    plan = P.AttentionPlan([0, 70], num_heads=2, num_kv_heads=2, head_dim=64, dtype=dtype)
    P.masked_attention(plan, q, k, v, out, 1.0)
    s = np.einsum("ihd,jhd->hij", q64, k64)
    first, second = np.sort(s, 2)[..., -1], np.sort(s, 2)[..., -2]
    clear = (first - second > 100).T
    best = s.argmax(2).T
    want = v64[best, np.arange(2)[None]]
    got = host(out)
    assert np.isfinite(got).all() and clear.mean() > 0.8
    rel = 12 * R.E32 if dtype == F32 else 2 * R.E16 * (1 + R.E16) + 12 * R.E32
    within(got[clear], want[clear], rel * np.abs(want[clear]))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_minus_infinity(dtype):
    """A row whose scores are all -inf has no weights; one -inf key has none."""
    q = torch.ones(2, 1, 16, dtype=dtype, device=DEV)
    k = torch.ones(3, 1, 16, dtype=dtype, device=DEV)
    v = torch.arange(48, dtype=torch.float32, device=DEV).view(3, 1, 16).to(dtype)
    k[1] = -math.inf
    out, lse = torch.empty_like(q), torch.empty(2, 1, device=DEV)
    plan = P.AttentionPlan([0, 2], [0, 3], num_heads=1, num_kv_heads=1, head_dim=16, dtype=dtype)
    P.masked_attention(plan, q, k, v, out, 1.0, lse=lse)
    np.testing.assert_allclose(host(out), np.broadcast_to((host(v)[0] + host(v)[2]) / 2, (2, 1, 16)),
                               rtol=2.0 ** -8)
    k[:] = -math.inf
    P.masked_attention(plan, q, k, v, out, 1.0, lse=lse)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_bits_do_not_change(dtype):
    """Repeated calls, and calls on another stream beside them, are equal bit for bit."""
    rng = np.random.default_rng(12)
    lens = [700, 90, 1, 333]
    o = offsets(lens)
    q, k, v = (normal(rng, (int(o[-1]), h, 128), dtype)[0] for h in (8, 2, 2))
    q1 = q[torch.from_numpy(o[:-1])].contiguous()
    for qq, qo in ((q, o), (q1, np.arange(5))):
        plan = P.AttentionPlan(qo, o, num_heads=8, num_kv_heads=2, head_dim=128, dtype=dtype)
        first = torch.empty_like(qq)
        P.masked_attention(plan, qq, k, v, first, 0.1)
        torch.cuda.synchronize()
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        outs = []
        for i in range(6):
            with torch.cuda.stream(side[i % 2]):
                outs.append(torch.empty_like(qq))
                P.masked_attention(plan, qq, k, v, outs[-1], 0.1)
        torch.cuda.synchronize()
        assert all(torch.equal(first, x) for x in outs)


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_of_several_threads(dtype):
    """Threads on streams of their own share a plan: every call's bits are the first one's."""
    rng = np.random.default_rng(17)
    o = offsets([500, 3, 210])
    plans = [P.AttentionPlan(o, num_heads=4, num_kv_heads=2, head_dim=64, dtype=dtype),
             P.AttentionPlan(np.arange(4), o, num_heads=4, num_kv_heads=2, head_dim=64, dtype=dtype)]
    q, k, v = (normal(rng, (int(o[-1]), h, 64), dtype)[0] for h in (4, 2, 2))
    want = [torch.empty_like(q) for _ in plans]
    for p, w in zip(plans, want):
        P.masked_attention(p, q, k, v, w, 0.1)
    torch.cuda.synchronize()

    def work(i):
        outs = []
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                outs.append(torch.empty_like(q))
                P.masked_attention(plans[i % 2], q, k, v, outs[-1], 0.1)
            torch.cuda.current_stream().synchronize()
        n = plans[i % 2].q_rows
        return all(torch.equal(x[:n], want[i % 2][:n]) for x in outs)

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(8)))


@pytest.mark.parametrize("dtype", TYPES)
def test_plan_let_go_behind_a_call(dtype):
    """Destroying a plan waits for the work that uses it."""
    rng = np.random.default_rng(18)
    n = 6000
    q, k, v = (normal(rng, (n, h, 128), dtype)[0] for h in (8, 2, 2))

    def call():
        plan = P.AttentionPlan([0, n], num_heads=8, num_kv_heads=2, head_dim=128, dtype=dtype,
                               causal=True)
        out = torch.empty_like(q)
        for _ in range(3):
            P.masked_attention(plan, q, k, v, out, 0.1)
        return out

    first, second = call(), call()
    torch.cuda.synchronize()
    assert torch.equal(first, second)


def test_attention_refuses_small_and_skew_workspaces():
    plan = P.AttentionPlan([0, 1], [0, 5000], num_heads=2, num_kv_heads=1, head_dim=64, dtype=F32)
    q, k = torch.zeros(1, 2, 64, device=DEV), torch.zeros(5000, 1, 64, device=DEV)
    size = plan.workspace_bytes
    assert size > 0
    room = torch.zeros(size + 16, dtype=torch.uint8, device=DEV)
    for bad in (room[:size - 1], room[1:size + 1], room[:0]):
        with pytest.raises(svl_amd.SvlError) as e:
            P.masked_attention(plan, q, k, k, torch.empty_like(q), 1.0, workspace=bad)
        assert e.value.kind == "Usage"
    P.masked_attention(plan, q, k, k, torch.empty_like(q), 1.0, workspace=room[:size])


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_in_a_graph(dtype):
    """Positions, rotation and attention captured twice, replayed together on two streams with
    eager calls between: each replay equals the eager run on its inputs."""
    seg = [(0, 0, 30, 0, 0, 0), (0, 1, 3, 8, 8, 2), (1, 1, 1, 16, 16, 1), (1, 0, 11, 0, 0, 0)]
    pp = P.PositionPlan(seg)
    n, hd = pp.tokens, 64
    o = np.array([0, 30 + 192, n])
    plans = [P.AttentionPlan(o, num_heads=4, num_kv_heads=2, head_dim=hd, dtype=dtype, causal=True),
             P.AttentionPlan(np.arange(3), o, num_heads=4, num_kv_heads=2, head_dim=hd, dtype=dtype)]
    axis, freq = axes_of(32, "mixed"), freqs(32)
    rng = np.random.default_rng(13)

    def layer(x, plan, ws):
        pos = torch.empty(n, 3, dtype=torch.int32, device=DEV)
        P.axis_positions(pp, pos)
        q, k = torch.empty_like(x[:, :4]), torch.empty_like(x[:, 4:6])
        P.rope_axes(x[:, :4], x[:, 4:6], pos, freq, axis, "half", q, k)
        out = torch.empty_like(q[:plan.q_rows])
        P.masked_attention(plan, q, k, x[:, 6:], out, 0.125, soft_cap=30.0, workspace=ws)
        return out

    x = [normal(rng, (n, 8, hd), dtype)[0] for _ in plans]
    ws = [torch.empty(max(p.workspace_bytes, 1), dtype=torch.uint8, device=DEV) for p in plans]
    graphs, outs = [], []
    for p, xx, w in zip(plans, x, ws):
        layer(xx, p, w)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(xx, p, w))
        graphs.append(g)
    side = [torch.cuda.Stream() for _ in graphs]
    for i in range(4):
        for xx in x:
            xx.copy_(normal(rng, xx.shape, dtype)[0])
        torch.cuda.synchronize()
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for p, xx, got in zip(plans, x, outs):
            assert torch.equal(layer(xx, p, None), got), i


@pytest.mark.parametrize("dtype", TYPES)
def test_operators_together(dtype):
    """A packed batch through positions, rotation and attention, as a layer uses them, against the
    64-bit form of the whole (each step from the values the step before it stored)."""
    seg = [(0, 0, 20, 0, 0, 0), (0, 1, 2, 6, 7, 1), (0, 0, 9, 0, 0, 0), (1, 1, 5, 4, 4, 3),
           (2, 0, 65, 0, 0, 0)]
    lens = [20 + 84 + 9, 80, 65]
    plan = P.PositionPlan(seg)
    rng = np.random.default_rng(14)
    nh, kv, hd = 3, 1, 256
    rows, r64 = normal(rng, (plan.tokens, nh + 2 * kv, hd), dtype)
    pos = torch.empty(plan.tokens, 3, dtype=torch.int32, device=DEV)
    P.axis_positions(plan, pos)
    np.testing.assert_array_equal(pos.cpu().numpy(), R.positions(seg))
    q, k, v = rows[:, :nh], rows[:, nh:nh + kv], rows[:, nh + kv:]
    axis, freq = axes_of(hd // 2, "runs"), freqs(hd // 2)
    P.rope_axes(q, k, pos, freq, axis, "axial", q, k)     # in place, in the fused rows
    for x, y in ((r64[:, :nh], q), (r64[:, nh:nh + kv], k)):
        want = R.rope(x, R.positions(seg), freq, axis, "axial")
        within(host(y), want, R.rope_bound(x, want, axis, "axial", dtype == BF16))
    o = offsets(lens)
    out = torch.empty_like(q)
    attn = P.AttentionPlan(o, num_heads=nh, num_kv_heads=kv, head_dim=hd, dtype=dtype, causal=True,
                           prefix=[40, 0, 5])
    P.masked_attention(attn, q, k, v, out, 1 / 16, soft_cap=50.0)
    want, _, bound, _ = R.attention(host(q), host(k), host(v), o, o, causal=True,
                                    prefix=[40, 0, 5], scale=1 / 16, cap=50.0, bf16=dtype == BF16)
    within(host(out), want, bound)


def test_attention_refuses_other_tensors():
    plan = P.AttentionPlan([0, 4], num_heads=2, num_kv_heads=1, head_dim=8, dtype=F32)
    q, k = torch.zeros(4, 2, 8, device=DEV), torch.zeros(4, 1, 8, device=DEV)
    out = torch.empty_like(q)
    s = torch.zeros(2, device=DEV)
    bad = [dict(q=q[:3]), dict(k=q), dict(v=k.bfloat16()), dict(out=out.cpu()),
           dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(slopes=s[:1]),
           dict(slopes=s.double()), dict(lse=torch.zeros(4, 3, device=DEV)),
           dict(lse=torch.zeros(4, 2, device=DEV, dtype=torch.float64)), dict(scale=math.nan),
           dict(scale=math.inf), dict(soft_cap=-1.0), dict(soft_cap=math.inf),
           dict(out=out[:1].expand(4, 2, 8)), dict(workspace=torch.zeros(4, device=DEV))]
    for change in bad:
        args = dict(q=q, k=k, v=k, out=out, scale=1.0)
        args.update(change)
        with pytest.raises(svl_amd.SvlError) as e:
            P.masked_attention(plan, **args)
        assert e.value.kind == "Usage", change
    with pytest.raises(svl_amd.SvlError) as e:
        P.AttentionPlan([0, 4], num_heads=2, num_kv_heads=1, head_dim=8, dtype=torch.float16)
    assert e.value.kind == "Unsupported"
