"""The paged 8-bit cache on the GPU (mmrs_paged_append, mmrs_paged_attend) against plain 64-bit
implementations (tests/paged_cases.py), at the sizes, masks and values where it can go wrong."""
from __future__ import annotations

import math

import pytest
import torch
from paged_cases import (D, NAN_CODE, Case, append64, attend64, attend_bounds, code_values, rope64, rope_tables)

pytestmark = pytest.mark.gpu


def check_attend(pkg, dev, c: Case, heads, dtype, window=0, sinks=0, q=None, scale=None, want_bounds=True):
    q = (c.randn(c.tokens, heads, D) * 1.5).to(dtype) if q is None else q
    cache, batch = c.cache(pkg, dev), c.batch(pkg, dev)
    lse = torch.full((c.tokens, heads), 7.0, device=dev)
    out = cache.attend(batch, q.to(dev), window=window, sinks=sinks, lse=lse, scale=scale)
    again = cache.attend(batch, q.to(dev), window=window, sinks=sinks, scale=scale)
    torch.cuda.synchronize()
    assert cache.status() == pkg.MMRS_OK
    assert torch.equal(out.view(torch.int16), again.view(torch.int16)), "two calls differ"
    ref, ref_lse, size, reach = attend64(c, q, D ** -0.5 if scale is None else scale, window, sinks)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(lse.isnan(), ref_lse.isnan())
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (out[empty] == 0).all()
    fine = ~ref_lse.isnan() & ~empty
    b_out, b_lse = attend_bounds(c, ref, size, reach, dtype)
    off = (out - ref).abs()[fine] - b_out[fine]
    assert off.numel() == 0 or off.max() <= 0, float(((out - ref).abs() / b_out)[fine].max())
    off = (lse - ref_lse).abs()[fine] - b_lse[fine]
    assert off.numel() == 0 or off.max() <= 0, float(((lse - ref_lse).abs() / b_lse)[fine].max())
    return out, lse


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group,kv", [(6, 8), (1, 3), (16, 1), (5, 2)])
def test_attend_single_tokens(pkg, dev, page, dtype, group, kv):
    c = Case([(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 300), (1, 1029)], page, kv, seed=page + group)
    c.spoil_unused()
    check_attend(pkg, dev, c, group * kv, dtype)


@pytest.mark.parametrize("group,kv", [(6, 2), (1, 2), (8, 1), (16, 1), (3, 1)])
@pytest.mark.parametrize("seqs", [[(5, 5), (2, 700), (1, 33), (4, 130)], [(8, 2000)], [(3, 3), (0, 50), (3, 64)]])
def test_attend_drafts(pkg, dev, group, kv, seqs):
    c = Case(seqs, 32, kv, seed=group)
    c.spoil_unused()
    check_attend(pkg, dev, c, group * kv, torch.bfloat16)


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("group,new", [(6, 6), (6, 8), (6, 9), (6, 11), (6, 16), (16, 3), (16, 4), (16, 6), (1, 33),
                                       (1, 48), (1, 49), (1, 64), (1, 65), (1, 96), (1, 97), (5, 9), (5, 10), (5, 20)])
def test_attend_rows_around_the_kernels_bounds(pkg, dev, page, group, new):
    """33 to 100 rows a KV head: two groups of the one kernel up to 48, one or both tiles of the other from there."""
    c = Case([(new, 400), (new, new), (1, 77), (new - 1, 1000)], page, 2, seed=page + new)
    c.spoil_unused()
    check_attend(pkg, dev, c, 2 * group, torch.float16)


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("group,kv", [(6, 2), (16, 1), (1, 2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_attend_tokens_drafts_and_prompts_together(pkg, dev, page, group, kv, window, sinks):
    """One call that both kernels serve; an empty sequence between them."""
    c = Case([(1, 500), (5, 310), (300, 450), (0, 20), (1, 1), (17, 17), (130, 130), (1, 900)], page, kv, seed=page + group)
    c.spoil_unused()
    check_attend(pkg, dev, c, group * kv, torch.bfloat16, window=window, sinks=sinks)


@pytest.mark.parametrize("new", [1, 5, 150])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_attend_negative_and_zero_scale(pkg, dev, new, scale):
    c = Case([(new, 333), (new, 190)], 32, 2, seed=new)
    check_attend(pkg, dev, c, 12, torch.float16, scale=scale)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group,kv,seqs", [(6, 2, [(129, 129), (300, 900)]), (1, 2, [(257, 1000), (1, 513)]),
                                           (8, 1, [(77, 400), (0, 9), (1, 1), (200, 201)]), (16, 1, [(64, 640)]),
                                           (5, 1, [(513, 700)])])
def test_attend_prompts(pkg, dev, page, dtype, group, kv, seqs):
    c = Case(seqs, page, kv, seed=page + group)
    c.spoil_unused()
    check_attend(pkg, dev, c, group * kv, dtype)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 3), (17, 16), (63, 100), (500, 4), (5000, 4)])
@pytest.mark.parametrize("seqs", [[(1, 1000), (1, 1), (1, 70)], [(4, 600), (2, 20)], [(200, 650), (33, 33)]])
def test_attend_window_and_sinks(pkg, dev, window, sinks, seqs):
    c = Case(seqs, 32, 2, seed=window + sinks)
    c.spoil_unused()
    check_attend(pkg, dev, c, 12, torch.float16, window=window, sinks=sinks)


@pytest.mark.parametrize("seqs", [[(1, 5000)], [(1, 20000), (1, 77)], [(3, 9000)], [(130, 4100)]])
def test_attend_long(pkg, dev, seqs):
    c = Case(seqs, 64, 2, seed=seqs[0][1])
    check_attend(pkg, dev, c, 12, torch.float16)


@pytest.mark.parametrize("new", [1, 4, 150])
def test_attend_pages_outside_the_pool(pkg, dev, new):
    """Positions of such pages are not seen; a row that sees nothing gives 0 and -infinity."""
    c = Case([(new, 400), (new, 200), (new, 333)], 16, 2, seed=new)
    c.table[0, 3:9] = -1
    c.table[1, :] = c.pages + 5
    c.table[2, 20] = 2 ** 31 - 1
    check_attend(pkg, dev, c, 12, torch.float16)
    # whole windows in such pages
    check_attend(pkg, dev, c, 12, torch.float16, window=20)


@pytest.mark.parametrize("new", [1, 3, 140])
def test_attend_nan_tokens_poison_only_rows_that_see_them(pkg, dev, new):
    c = Case([(new, 300), (new, 500)], 32, 2, seed=new)
    for b, j, h in ((0, 299, 0), (1, 50, 1)):
        pid = c.table[b, j // 32]
        c.k[pid, h, j % 32] = NAN_CODE
        c.v[pid, h, j % 32] = 0
    out, _ = check_attend(pkg, dev, c, 12, torch.bfloat16)
    assert out.isnan().any() and not out.isnan().all()
    check_attend(pkg, dev, c, 12, torch.bfloat16, window=30)


@pytest.mark.parametrize("new", [2, 150])
@pytest.mark.parametrize("level", [2.0 ** -40, 2.0 ** 12])
def test_attend_scales_of_any_size(pkg, dev, new, level):
    """Pages whose scales differ by many powers of two, and zero scales."""
    c = Case([(new, 700)], 32, 2, seed=new)
    c.vs[::2] *= level
    c.vs[1] = 0.0
    c.ks[3] = 0.0
    check_attend(pkg, dev, c, 12, torch.float16)


@pytest.mark.parametrize("new", [1, 160])
@pytest.mark.parametrize("size", [1e-30, 3e4])
def test_attend_query_sizes(pkg, dev, new, size):
    c = Case([(new, 333)], 64, 2, seed=new)
    q = (c.randn(c.tokens, 12, D) * size).to(torch.bfloat16)
    check_attend(pkg, dev, c, 12, torch.bfloat16, q=q, scale=0.02 / size)


@pytest.mark.parametrize("new", [1, 150])
def test_attend_strided_queries_on_another_stream(pkg, dev, new):
    c = Case([(new, 333), (new, 190)], 64, 2, seed=new)
    wide = c.randn(c.tokens, 20, D).to(torch.float16)
    q = wide[:, 4:16]
    ref, _, size, reach = attend64(c, q)
    wide_dev, cache, batch = wide.to(dev), c.cache(pkg, dev), c.batch(pkg, dev)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    out = torch.empty(c.tokens, 12, D, dtype=torch.float16, device=dev)
    cache.workspace(2, c.tokens, 12)
    torch.cuda.synchronize()
    cache.attend(batch, wide_dev[:, 4:16], out=out, stream=stream)
    stream.synchronize()
    bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
    assert ((out.cpu().double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("new", [1, 40])
def test_first_call_on_another_stream(pkg, dev, new):
    """Workspace and outputs are made on the stream of the call, not on the current one, which is busy here."""
    c = Case([(new, 333), (new, 190)], 64, 2, seed=new)
    q = c.randn(c.tokens, 12, D).to(torch.float16)
    ref, _, size, reach = attend64(c, q)
    q_dev, cache, batch = q.to(dev), c.cache(pkg, dev), c.batch(pkg, dev)
    stream, big = torch.cuda.Stream(), torch.empty(1 << 28, device=dev)
    torch.cuda.synchronize()
    for _ in range(20):
        big.normal_()
    out = cache.attend(batch, q_dev, stream=stream)
    stream.synchronize()
    with torch.cuda.stream(stream):
        got = out.cpu().double()
    bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
    assert ((got - ref).abs() <= bound).all() and cache.status() == pkg.MMRS_OK


def test_attend_same_call_with_looser_bounds(pkg, dev):
    """max_q and max_len are bounds: a captured call serves shorter lengths with the same result."""
    c = Case([(2, 600), (1, 90)], 32, 2, seed=3)
    q = c.randn(c.tokens, 12, D).to(torch.float16)
    ref, _, size, reach = attend64(c, q)
    c.table = torch.cat([c.table, torch.full((2, 100), -1, dtype=torch.int32)], 1).contiguous()
    bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
    cache = c.cache(pkg, dev)
    for max_q, max_len in ((2, 600), (5, 3000), (64, 3000)):
        out = cache.attend(c.batch(pkg, dev, max_q=max_q, max_len=max_len), q.to(dev))
        assert ((out.cpu().double() - ref).abs() <= bound).all(), (max_q, max_len)


def test_attend_graph_replay_with_other_lengths(pkg, dev):
    c = Case([(1, 900), (1, 500)], 64, 2, seed=8)
    q = c.randn(c.tokens, 12, D).to(torch.float16)
    cache, batch, q_dev = c.cache(pkg, dev), c.batch(pkg, dev), q.to(dev)
    out = torch.empty_like(q_dev)
    cache.attend(batch, q_dev, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(batch, q_dev, out=out)
    for lens in ([900, 500], [3, 499], [64, 1]):
        batch.t[1].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c.seqs = [(1, n) for n in lens]
        ref, _, size, reach = attend64(c, q)
        bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
        assert ((out.cpu().double() - ref).abs() <= bound).all(), lens


def test_attend_and_append_past_two_gigabytes(pkg, dev):
    """Codes at byte offsets past 2^31 (and page rows past 2^24)."""
    pages, page, kv = 36000, 64, 8
    c = Case([(1, 200), (150, 150)], page, kv, seed=5)
    q = c.randn(c.tokens, 48, D).to(torch.float16)
    ref, _, size, reach = attend64(c, q)
    cache = pkg.PagedKvCache(pages, dev, kv_heads=kv, page_size=page)
    at = pages - c.pages
    for big, small in ((cache.k, c.k), (cache.v, c.v)):
        big.view(torch.uint8)[at:].copy_(small.to(dev))
    cache.k_scale[at:] = c.ks.to(dev)
    cache.v_scale[at:] = c.vs.to(dev)
    c.table = torch.where(c.table >= 0, c.table + at, c.table)
    out = cache.attend(c.batch(pkg, dev), q.to(dev))
    bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
    assert ((out.cpu().double() - ref).abs() <= bound).all()
    cos, sin = (x.to(dev) for x in rope_tables(64, 300))
    k = c.randn(c.tokens, kv, D).to(dev)
    cache.append(c.batch(pkg, dev), None, k, k, cos, sin)
    last = cache.v.view(torch.uint8)[int(c.table[0, 3]), :, 199 % 64].cpu()
    got = code_values(last) * cache.v_scale[int(c.table[0, 3])].cpu().double()[:, None]
    assert ((got - k[0].cpu().double()).abs() <= 2.0 ** -4 * k[0].cpu().double().abs() + 2.0 ** -10).all()


def check_append(pkg, dev, c: Case, heads, dtype, rope_dim, k=None, v=None, out_dtype=None):
    width = (heads + 2 * c.kv) * D
    wide = (c.randn(c.tokens, width) * torch.exp(c.randn(1, width))).to(dtype)
    q = wide[:, :heads * D].unflatten(1, (heads, D))
    k = wide[:, heads * D:(heads + c.kv) * D].unflatten(1, (c.kv, D)) if k is None else k
    v = wide[:, (heads + c.kv) * D:].unflatten(1, (c.kv, D)) if v is None else v
    cos, sin = rope_tables(rope_dim, c.max_len + 1)
    pos = torch.cat([torch.arange(n - m, n) for m, n in c.seqs])
    want = append64(c, k, v, cos, sin)
    cache, batch = c.cache(pkg, dev), c.batch(pkg, dev)
    wd = wide.to(dev)
    q_out = torch.empty(c.tokens, heads, D, dtype=out_dtype, device=dev) if out_dtype else None
    args = (wd[:, :heads * D].unflatten(1, (heads, D)), k.to(dev), v.to(dev), cos.to(dev), sin.to(dev))
    got_q = cache.append(batch, *args, q_out=q_out).clone()
    torch.cuda.synchronize()
    first = [x.clone() for x in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    # queries: f32 products and sums (three roundings), then one rounding to 16 bits
    ref_q = rope64(q, cos, sin, pos)
    unit = 2.0 ** -8 if got_q.dtype == torch.bfloat16 else 2.0 ** -11
    half = rope_dim // 2
    pair = torch.zeros_like(ref_q)
    pair[..., :rope_dim] = (q[..., :half].abs().double() + q[..., half:rope_dim].abs().double()).repeat(1, 1, 2)
    assert ((got_q.cpu().double() - ref_q).abs() <= unit * ref_q.abs() + 2.0 ** -22 * pair + 2.0 ** -25).all()
    for codes, scale, (val, sc, new, broken, free), is_key, before in (
            (first[0], first[2], want[0], True, (c.k, c.ks)), (first[1], first[3], want[1], False, (c.v, c.vs))):
        codes, scale = codes.cpu(), scale.cpu().double()
        amax_edge = 2.0 ** -20  # a largest value this near 448 s may fall on either side in 32 bits
        bad = scale != sc
        if bad.any():
            most = torch.where(new[..., None] & ~broken[..., None], val, torch.zeros_like(val)).abs().amax((2, 3))
            near = ((most / (448 * sc)) - 1).abs() < amax_edge
            near |= ((most / (224 * sc)) - 1).abs() < amax_edge
            assert (near | ~bad).all()
        got = code_values(codes) * scale[:, :, None, None]
        # a code: half a step of three mantissa bits (2^-4 of the value) or of the subnormals (2^-10 scale)
        tol = (2.0 ** -4 + 2.0 ** -12) * val.abs() + 2.0 ** -10 * scale[:, :, None, None] * (1 + 2.0 ** -12)
        ok = (got - val).abs() <= tol
        live = ~(broken | free)[..., None].expand_as(ok)
        assert ok[live].all(), float((got - val).abs()[live].max())
        if broken.any():
            dead = codes[broken]
            assert (dead & 0x7F == NAN_CODE).all() if is_key else (code_values(dead) == 0).all()
        untouched = ~new.any(2)
        assert torch.equal(codes[untouched], before[0][untouched])
        assert torch.equal(scale[untouched], before[1].double()[untouched])
    cache.append(batch, *args, q_out=q_out)
    torch.cuda.synchronize()
    for x, y in zip(first, (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)):
        assert torch.equal(x, y), "a second call with the same arguments changed the cache"
    return cache


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rope_dim", [64, 0, 128, 6, 36])
def test_append(pkg, dev, page, dtype, rope_dim):
    c = Case([(1, 1), (1, 400), (5, 131), (130, 130), (70, 250), (0, 10), (3, 65)], page, 2, seed=page + rope_dim)
    check_append(pkg, dev, c, 12, dtype, rope_dim)


@pytest.mark.parametrize("heads,kv", [(48, 8), (1, 1), (5, 5), (32, 4)])
def test_append_heads(pkg, dev, heads, kv):
    c = Case([(1, 900), (9, 77), (1, 64), (1, 65)], 64, kv, seed=heads)
    check_append(pkg, dev, c, heads, torch.float32, 64, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("level", [2.0 ** -30, 1.0, 2.0 ** 20])
def test_append_rescales_older_codes(pkg, dev, level):
    """Pages whose older codes have smaller (larger) scales than the new tokens need."""
    c = Case([(1, 50), (3, 100), (2, 40)], 64, 2, seed=1, level=level)
    check_append(pkg, dev, c, 2, torch.float32, 64)


def test_append_not_finite_and_zero_tokens(pkg, dev):
    c = Case([(6, 70), (4, 4), (40, 80)], 32, 2, seed=4)
    k, v = c.randn(c.tokens, 2, D), c.randn(c.tokens, 2, D)
    k[0, 0, 5], v[3, 1, 0], k[7, 1, 127], v[12, 0, 64] = math.nan, math.inf, -math.inf, math.nan
    k[6:10, 0], v[6:10, 0] = 0.0, 0.0  # a sequence whose first tokens are all zero
    cache = check_append(pkg, dev, c, 2, torch.float32, 64, k=k, v=v)
    assert not cache.k_scale.isnan().any() and not cache.v_scale.isnan().any()


def test_append_skips_pages_outside_the_pool(pkg, dev):
    c = Case([(40, 100), (1, 64)], 16, 2, seed=6)
    c.table[0, 4] = -1
    c.table[1, 3] = c.pages
    check_append(pkg, dev, c, 2, torch.float16, 64)


def test_tokens_one_by_one_read_back_like_a_prompt(pkg, dev):
    """Appending token by token and attending gives what one call for all of them gives, up to what the
    codes' scales differ by on the way."""
    n, kv, heads, page = 70, 2, 12, 32
    c = Case([(n, n)], page, kv, seed=9)
    q, k, v = (c.randn(n, h, D).to(torch.float16) for h in (heads, kv, kv))
    cos, sin = (x.to(dev) for x in rope_tables(64, n + 1))
    whole, steps = c.cache(pkg, dev), c.cache(pkg, dev)
    table = c.table.to(dev)
    batch = c.batch(pkg, dev)
    a = whole.attend(batch, whole.append(batch, q.to(dev), k.to(dev), v.to(dev), cos, sin))
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    for i in range(n):
        one = pkg.PagedBatch(cu, torch.tensor([i + 1], dtype=torch.int32, device=dev), table, max_q=1, max_len=n)
        rot = steps.append(one, *(x[i:i + 1].to(dev) for x in (q, k, v)), cos, sin)
        b = steps.attend(one, rot)
        # scores move by at most the keys' rounding (2^-4 of 128 products' root sum): well under 0.2 of the values
        assert (a[i:i + 1].float() - b.float()).norm() <= 0.1 * a[i:i + 1].float().norm()
    pages = c.table[0, :3].long()
    assert torch.equal(whole.k_scale[pages], steps.k_scale[pages])
    assert torch.equal(whole.k.view(torch.uint8)[pages[:2]], steps.k.view(torch.uint8)[pages[:2]]) or \
        (whole.k.float()[pages[:2]] - steps.k.float()[pages[:2]]).abs().max() <= 2.0 ** -9


def test_nothing_to_do(pkg, dev):
    cache = pkg.PagedKvCache(4, dev, kv_heads=2, page_size=16)
    cu = torch.zeros(2, dtype=torch.int32, device=dev)
    lens = torch.tensor([5], dtype=torch.int32, device=dev)
    batch = pkg.PagedBatch(cu, lens, torch.zeros(1, 1, dtype=torch.int32, device=dev), max_q=1, max_len=16)
    q = torch.empty(0, 12, D, dtype=torch.float16, device=dev)
    k = torch.empty(0, 2, D, dtype=torch.float16, device=dev)
    cos, sin = (x.to(dev) for x in rope_tables(64, 16))
    assert cache.append(batch, q, k, k, cos, sin).shape == (0, 12, D)
    assert cache.attend(batch, q).shape == (0, 12, D)
