"""The serving operators where values are not finite, where a call is refused half way through a decoding
round, and at sizes that reach the paths of large launches. Tolerances: tests/serving_reference.py."""
import pytest
import torch

from tests.serving_reference import close
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
