"""The serving operators where values are not finite, where a call is refused half way through a decoding
round, and at sizes that reach the paths of large launches. Tolerances: tests/serving_reference.py."""
import pytest
import torch

from tests.serving_reference import attention, close
from tests.test_gpu_serving import BF, DEV, F32, SCALE, i32, paged_inputs, paged_reference, prompt_inputs, \
    prompt_reference, token_kv

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def quickest(f, n=3):
    """Milliseconds of the fastest of n calls after a warm-up."""
    f()
    best = INF
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


# ---------------------------------------------------------------- scores of minus infinity
@pytest.mark.parametrize("dtype", [BF, F32])
def test_every_score_minus_infinity_is_not_an_empty_row(dtype):
    """A softmax over scores that are all -inf has no value, whether one chunk holds them or many; a sequence
    without a page is zero all the same."""
    from respect_b200.kernels import paged_attention, prompt_attention
    lens = [1, 40, 700, 700, 500, 300, 130]
    q, k, v, table, seqs = paged_inputs(51, lens, 8, 2, 16, dtype)
    q[..., 0] = q[..., 0].abs() + 1
    ref, tol = paged_reference(q, seqs)
    for b, n in enumerate(lens):
        first = 0 if b != 3 else 350                        # sequence 3: its first half stays as it is
        if b == 5:
            continue                                        # as it is throughout
        for j in range(first, n):
            k[table[b, j // 16], :, j % 16, 0] = -INF
    table[4, :5], table[4, 9] = -1, -1                      # pages missing before and among them
    table[6] = -1
    ref[[0, 1, 2, 4]] = NAN
    ref[6] = 0
    ref[3], tol[3] = (x[0] for x in paged_reference(q[3:4], [(seqs[3][0][:350], seqs[3][1][:350])]))
    y = paged_attention(q, k, v, table, i32(lens))
    close(y, ref, tol)
    kk = seqs[1][0].clone()
    kk[:, :, 0] = -INF
    p = prompt_attention(q[1:2].expand(40, -1, -1), kk, seqs[1][1], i32([0, 40]))
    assert torch.equal(p[39].isnan(), y[1].isnan()) and bool(p.isnan().all())


# ---------------------------------------------------------------- bad values beside a key that takes everything
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,bad,best", [(40, 3, 30), (40, 30, 3), (300, 5, 20), (300, 20, 5), (300, 5, 290), (300, 290, 5)])
def test_a_nan_beside_a_dominating_key_stays(dtype, n, bad, best):
    """An attended NaN shows wherever the key lies that takes all the weight: before it, after it, in the same
    chunk or tile or in another."""
    from respect_b200.kernels import paged_attention, prompt_attention
    q, k, v, table, seqs = paged_inputs(52, [n], 8, 2, 16, dtype)
    q[..., 0] = 40.0
    k[table[0, best // 16], :, best % 16, 0] = 40.0         # a score of 1600 / sqrt(128): the others weigh 2^-200
    v[table[0, bad // 16], 1, bad % 16, 9] = NAN
    # the plain value of the other entries: V of the dominating key, up to weights of 2^-180
    ref, tol = paged_reference(q, [(seqs[0][0][best:best + 1], seqs[0][1][best:best + 1])])
    ref[0, 4:, 9] = NAN
    close(paged_attention(q, k, v, table, i32([n])), ref, tol)
    kk, vv = seqs[0][0].clone(), seqs[0][1].clone()
    kk[best, :, 0], vv[bad, 1, 9] = 40.0, NAN
    y = prompt_attention(q.expand(n, -1, -1), kk, vv, i32([0, n]))
    ref, tol = ref.expand(n, -1, -1).clone(), tol * (1 if dtype == F32 else 2)   # bf16 prompts: one part of P, 2^-8 more
    ref[:bad, 4:, 9] = seqs[0][1][best, 1, 9].double()
    close(y[max(best, bad):], ref[max(best, bad):], tol.expand(n, -1, -1)[max(best, bad):])
    if best < bad:
        close(y[best:bad], ref[best:bad], tol.expand(n, -1, -1)[best:bad])


# ---------------------------------------------------------------- a round that cannot be served
def test_commit_takes_no_page_that_another_sequence_holds():
    """A fork, a pool without a free page, and a round of reserve, write and commit without a look at the
    status in between: nothing grows. After room is made the same round goes through."""
    from respect_b200.decoding.kv_pages import PagedCacheError, PagedKVCache
    cache = PagedKVCache(1, 2, 5, 16, 4, dtype=F32)
    cache.reserve([0, 3], [37, 32])
    cache.write(*token_kv(cache, list(range(69))), [0, 3], [0, 37, 69])
    cache.commit([0, 3], [37, 32])
    cache.fork([0], [1])
    cache.check()
    before = [t.clone() for t in (cache.store, cache.table, cache.lengths, cache.held, cache.refs)]
    seqs, ones = i32([1, 0]), i32([1, 1])
    new = token_kv(cache, [101, 100])
    cache.reserve(seqs, ones)
    cache.write(*new, seqs)
    cache.commit(seqs, ones)
    with pytest.raises(PagedCacheError, match="free pages"):
        cache.check()
    for a, b in zip(before, (cache.store, cache.table, cache.lengths, cache.held, cache.refs)):
        assert torch.equal(a, b)
    cache.commit([0], [1])                                  # alone, too
    with pytest.raises(PagedCacheError, match="another sequence holds"):
        cache.check()
    cache.commit([0, 1], [0, 0])                            # nothing asked: nothing refused
    cache.check()
    cache.free([3])
    cache.reserve(seqs, ones)
    cache.write(*new, seqs)
    cache.commit(seqs, ones)
    cache.check()
    assert cache.lengths.tolist() == [38, 38, 0, 0]
    for s, t in ((0, 100), (1, 101)):
        k, v = token_kv(cache, list(range(37)) + [t])
        page = cache.table[s].long()[torch.arange(38, device=DEV) // 16]
        assert torch.equal(cache.store[0, 0, page, :, torch.arange(38, device=DEV) % 16], k[0])
        assert torch.equal(cache.store[0, 1, page, :, torch.arange(38, device=DEV) % 16], v[0])


def test_commit_needs_its_pages():
    """A page missing from the table refuses the commit; a long commit looks at every page it covers."""
    from respect_b200.decoding.kv_pages import PagedCacheError, PagedKVCache
    cache = PagedKVCache(1, 1, 300, 2, 3, dtype=F32, head_dim=8)
    cache.reserve([0, 1], [400, 20])
    for at in (0, 77, 199):
        page = cache.table[0, at].item()
        cache.table[0, at] = -1
        cache.commit([1, 0], [20, 400])
        with pytest.raises(PagedCacheError, match="another sequence holds"):
            cache.check()
        cache.table[0, at] = page
        cache.refs[page] = 2
        cache.commit([0], [400])
        with pytest.raises(PagedCacheError, match="another sequence holds"):
            cache.check()
        cache.refs[page] = 1
    assert cache.lengths.tolist() == [0, 0, 0]
    cache.table[0, 199] = -1
    cache.commit([1, 0], [20, 398])                         # up to the missing page
    cache.check()
    assert cache.lengths.tolist() == [398, 20, 0]


# ---------------------------------------------------------------- scales of zero and below
def test_prompt_scales_of_zero_and_below_cost_no_more():
    """fp32: the same kernel at the same speed (and right, in a prompt of several tiles)."""
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(53, [1500, 333], 4, 1, F32)
    cu_t = i32(cu)
    plain = quickest(lambda: prompt_attention(q, k, v, cu_t))
    for scale in (-SCALE, 0.0, -0.25):
        close(prompt_attention(q, k, v, cu_t, sm_scale=scale), *prompt_reference(q, k, v, cu, scale))
        assert quickest(lambda: prompt_attention(q, k, v, cu_t, sm_scale=scale)) < 3 * plain + 0.05


# ---------------------------------------------------------------- values that are not finite, in prompts
def with_bad_entries(ref, cu, groups, bad):
    """A result with V entries (token, kv head, dim, value) added whose weights are not zero."""
    ref = ref.clone()
    for token, head, dim, value in bad:
        end = min(c for c in cu if c > token)
        ref[token:end, head * groups:(head + 1) * groups, dim] += value
    return ref


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,HK,lens", [(28, 4, [300, 1, 200, 90]), (16, 16, [700, 129, 1]), (64, 1, [40, 150]), (8, 1, [257, 31])])
def test_prompt_bad_values_at_every_place(dtype, H, HK, lens):
    """Infinities and NaN in V, several in a tile, on tiles' edges and in the first and last token: only the
    rows that attend to one show it, in its dim; the others keep their bits."""
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(61, lens, H, HK, dtype)
    clean = prompt_attention(q, k, v, i32(cu))
    ref, tol = prompt_reference(q, k, v, cu)
    last = cu[-1] - 1
    for case in ([(0, 0, 3, INF), (5, HK - 1, 127, NAN), (17, 0, 64, -INF), (18, 0, 64, INF)],
                 [(last, 0, 0, INF), (last, HK - 1, 63, NAN), (last - 1, 0, 0, -INF), (cu[1], 0, 8, -INF)],
                 [(t, t % HK, t % 128, (INF, -INF, NAN)[t % 3]) for t in range(last + 1)][::9],
                 [(t, 0, 40, INF) for t in (30, 31, 32, 33, 34)] + [(last - 3, 0, 40, -INF)]):
        v2, zero = v.clone(), v.clone()
        for token, head, dim, value in case:
            v2[token, head, dim], zero[token, head, dim] = value, 0
        y = prompt_attention(q, k, v2, i32(cu))
        want, tol2 = prompt_reference(q, k, zero, cu)
        close(y, with_bad_entries(want, cu, H // HK, case), tol2)
        untouched = with_bad_entries(torch.zeros_like(ref), cu, H // HK, [(t, h, d, 1.0) for t, h, d, _ in case]) == 0
        if dtype == BF:
            assert torch.equal(y[untouched], clean[untouched])
        assert torch.equal(prompt_attention(q, k, v2, i32(cu)).isnan(), y.isnan())
    # scores of -inf: such a key weighs nothing; the first token of a prompt has nothing else
    k2, q2 = k.clone(), q.clone()
    q2[..., 0] = q2[..., 0].abs() + 1
    for token in (cu[1], 20, last):
        k2[token, :, 0] = -INF
    # their weights are exactly zero on both sides, so what is left is attention over the other keys,
    # and its bound (the bound over all keys is infinite: it counts |q| |k|)
    want, tol2 = torch.full_like(ref, NAN), torch.zeros_like(tol)
    for a, b in zip(cu, cu[1:]):
        mask = torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).tril()
        mask &= (k2[a:b, 0, 0] != -INF)[None]
        some = mask.any(1)
        o, t = attention(q2[a:b], k2[a:b], v[a:b], mask, SCALE, 2.0 ** -8 if dtype == BF else 0.0)
        want[a:b][some], tol2[a:b][some] = o[some], t[some]
    close(prompt_attention(q2, k2, v, i32(cu)), want, tol2)


@pytest.mark.parametrize("dtype,H,n", [(BF, 4, 20000), (BF, 2, 150000), (F32, 4, 20000)])
def test_prompt_bad_values_cost_little(dtype, H, n):
    """A NaN that nearly every row of a long prompt attends to, and infinities further on: right, and within a
    small factor of the call without (fp32 goes over infinities a second time; rows settled one by one and key by
    key took hundreds of times as long)."""
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(62, [n], H, 1, dtype)
    cu = i32(cu)
    clean = prompt_attention(q, k, v, cu)
    plain = quickest(lambda: prompt_attention(q, k, v, cu))
    v = v.clone()
    v[3, 0, 5], v[n // 2, 0, 7], v[n - 70, 0, 9] = NAN, INF, -INF
    y = prompt_attention(q, k, v, cu)
    assert bool(y[3:, :, 5].isnan().all())
    assert bool((y[n // 2:, :, 7] == INF).all()) and bool((y[n - 70:, :, 9] == -INF).all())
    same = torch.ones_like(y, dtype=torch.bool)
    same[3:, :, 5], same[n // 2:, :, 7], same[n - 70:, :, 9] = False, False, False
    if dtype == BF:
        assert torch.equal(y[same], clean[same])
    else:
        assert bool(((y - clean).abs()[same] <= 1e-5).all())
    assert quickest(lambda: prompt_attention(q, k, v, cu)) < (3 if dtype == BF else 6) * plain + 0.1
