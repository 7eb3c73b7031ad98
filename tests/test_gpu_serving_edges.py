"""The serving operators where values are not finite, where a call is refused half way through a decoding
round, and at sizes that reach the paths of large launches. Tolerances: tests/serving_reference.py."""
import pytest
import torch

from tests import test_gpu_serving as base
from tests.serving_reference import attention, close
from tests.test_gpu_serving import BF, DEV, F32, SCALE, gen, i32, paged_inputs, paged_reference, prompt_inputs, \
    prompt_reference, randn, token_kv

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


# ---------------------------------------------------------------- sizes of large launches
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ps", [16, 24])
def test_paged_warps_that_take_several_chunks(dtype, ps):
    """Enough chunks in one call that a warp takes several of them: every row has the bits of a call of its
    own, in which a warp takes one."""
    from respect_b200.kernels import paged_attention
    lens = [2500, 1, 700, 2047, 130, 0]
    q, k, v, table, seqs = paged_inputs(54, lens, 16, 8, ps, dtype)
    ref, tol = paged_reference(q, seqs)
    pick = [i % 6 for i in range(96)]                       # 96 x 8 heads x 40 chunks (bf16) or 79 (fp32)
    y = paged_attention(q[pick], k, v, table, i32(lens), seqs=i32(pick))
    for row, i in enumerate(pick):
        if row < 6:
            close(y[i], ref[i], tol[i])
            assert torch.equal(paged_attention(q[i:i + 1], k, v, table, i32(lens), seqs=i32([i]))[0], y[i])
        else:
            assert torch.equal(y[row], y[i])


@pytest.mark.parametrize("H,HK,lens", [(16, 16, [6000, 300, 1, 2900]), (32, 8, [2500, 0, 6100, 33, 700]), (28, 4, [4100, 3000])])
def test_prompt_blocks_with_several_items_and_bands(H, HK, lens):
    """More work items than blocks (three and more a block) and prompts longer than a band of tiles."""
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(55 + H, lens, H, HK, BF)
    y = prompt_attention(q, k, v, i32(cu))
    close(y, *prompt_reference(q, k, v, cu))
    for a, b in zip(cu, cu[1:]):
        assert torch.equal(prompt_attention(q[a:b], k[a:b], v[a:b], i32([0, b - a])), y[a:b])


@pytest.mark.parametrize("tokens,layers", [(700, 8), (801, 28)])
def test_page_writes_of_several_layers_a_warp(tokens, layers):
    from respect_b200.decoding.kv_pages import PagedKVCache
    cache = PagedKVCache(layers, 2, 150, 16, 2, dtype=F32, head_dim=20)
    cut = tokens // 3
    cache.reserve([1, 0], [cut, tokens - cut])
    k, v = token_kv(cache, list(range(tokens)))
    cache.write(k, v, [1, 0], [0, cut, tokens])
    cache.commit([1, 0], [cut, tokens - cut])
    cache.check()
    for s, a, b in ((1, 0, cut), (0, cut, tokens)):
        pos = torch.arange(b - a, device=DEV)
        page, slot = cache.table[s].long()[pos // 16], pos % 16
        assert torch.equal(cache.store[:, 0][:, page, :, slot].transpose(0, 1), k[:, a:b])
        assert torch.equal(cache.store[:, 1][:, page, :, slot].transpose(0, 1), v[:, a:b])


def test_reserve_looks_through_a_large_pool():
    """More pages than one look of the planning block: the lowest free ones, in list order."""
    from respect_b200.decoding.kv_pages import PagedKVCache
    pages = 9001
    cache = PagedKVCache(1, 1, pages, 1, 4, dtype=F32, head_dim=4)
    free = torch.rand(pages, device=DEV, generator=gen(56)) < 0.6
    cache.refs.copy_(torch.where(free, 0, 1))
    low = free.nonzero()[:, 0].tolist()
    counts = [1, 2500, 0, 2600]
    cache.reserve([2, 0, 1, 3], counts)
    cache.check()
    at = 0
    for s, n in zip([2, 0, 1, 3], counts):
        assert cache.table[s, :n].tolist() == low[at:at + n] and bool((cache.table[s, n:] == -1).all())
        at += n
    assert cache.refs.nonzero()[:, 0].tolist() == sorted(low[:at] + (~free).nonzero()[:, 0].tolist())


def test_compact_of_long_paths():
    """Paths longer than the tokens a block looks up at a time."""
    from respect_b200.decoding.kv_pages import PagedKVCache
    cache = PagedKVCache(2, 2, 100, 16, 2, dtype=F32)
    cache.reserve([0, 1], [9, 500])
    cache.write(*token_kv(cache, list(range(509))), [0, 1], [0, 9, 509])
    path = sorted(torch.randperm(500, generator=torch.Generator().manual_seed(57))[:300].tolist())
    cache.compact([1, 0], [path, [0, 4, 8]], [300, 3])
    cache.check()
    assert cache.lengths.tolist() == [3, 300]
    for s, tokens in ((1, [9 + t for t in path]), (0, [0, 4, 8])):
        pos = torch.arange(len(tokens), device=DEV)
        page, slot = cache.table[s].long()[pos // 16], pos % 16
        k, v = token_kv(cache, tokens)
        assert torch.equal(cache.store[:, 0][:, page, :, slot].transpose(0, 1), k)
        assert torch.equal(cache.store[:, 1][:, page, :, slot].transpose(0, 1), v)


@pytest.mark.parametrize("ps,pages,layers,heads,dim", [(16, 30, 2, 3, 128), (5, 70, 3, 1, 8)])
def test_page_operations_follow_the_model_in_bf16(monkeypatch, ps, pages, layers, heads, dim):
    """The model test with values that bf16 holds exactly: a token's number in digits of base 16."""
    def digits(cache, tokens):
        t = torch.tensor(tokens, device=DEV, dtype=torch.int64).reshape(1, -1, 1, 1)
        part = torch.arange(cache.layers * cache.kv_heads, device=DEV).reshape(cache.layers, 1, cache.kv_heads, 1)
        d = torch.arange(cache.head_dim, device=DEV)
        k = ((t >> (d % 4 * 4) & 15) + 16 * (part % 16)).to(cache.dtype)
        return k, -k - 1
    monkeypatch.setattr(base, "token_kv", digits)
    base.test_page_operations_follow_the_model(ps, pages, BF, layers, heads, dim)


def test_page_operations_past_32_bits():
    """Pages whose elements lie beyond 2^31: written, copied for a fork, compacted and given back."""
    from respect_b200.decoding.kv_pages import PagedKVCache
    pages, low = 70000, 69980
    store = torch.empty(1, 2, pages, 4, 64, 128, device=DEV, dtype=BF)      # 4.6e9 elements
    z = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)
    refs = z(pages)
    refs[:low] = 1
    cache = PagedKVCache.from_state(store, z(3, 8) - 1, z(3), z(3), refs)
    k, v = randn(gen(58), 2, 1, 300, 4, 128, dtype=BF)
    cache.reserve([2], [100])
    cache.write(k[:, :100], v[:, :100], [2], [0, 100])
    cache.commit([2], [100])
    cache.fork([2], [0])
    cache.reserve([0], [200])                                  # copies the last page
    cache.write(k[:, 100:], v[:, 100:], [0], [0, 200])
    path = list(range(1, 200, 3))
    cache.compact([0], [path], [len(path)])
    cache.check()
    assert cache.table[2, :2].tolist() == [low, low + 1] and cache.table[0, :2].tolist() == [low, low + 2]
    for s, tokens in ((2, list(range(100))), (0, list(range(100)) + [100 + t for t in path])):
        pos = torch.arange(len(tokens), device=DEV)
        page, slot = cache.table[s].long()[pos // 64], pos % 64
        assert torch.equal(store[0, 0][page, :, slot], k[0, tokens]) and torch.equal(store[0, 1][page, :, slot], v[0, tokens])
    cache.free([0, 2])
    assert bool((refs[:low] == 1).all()) and not bool(refs[low:].any())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_prompts(dtype):
    """Thousands of prompts of a few tokens, many of them empty."""
    from respect_b200.kernels import prompt_attention
    lens = torch.randint(0, 6, (3000,), generator=torch.Generator().manual_seed(59)).tolist()
    lens[1700] = 200
    q, k, v, cu = prompt_inputs(59, lens, 8, 2, dtype, before=3, behind=2)
    y = prompt_attention(q, k, v, i32(cu))
    T = q.shape[0]
    owner = torch.bucketize(torch.arange(T, device=DEV), i32(cu), right=True)      # 0: before, 3001: behind
    mask = (owner[:, None] == owner[None]) & torch.ones(T, T, dtype=torch.bool, device=DEV).tril()
    mask[owner == 0], mask[owner == 3001] = False, False
    for r in range(0, T, 1024):
        close(y[r:r + 1024], *attention(q[r:r + 1024], k, v, mask[r:r + 1024], SCALE, 2.0 ** -8 if dtype == BF else 0.0))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_paged_wide_groups_and_pages(dtype):
    """Groups past a block's sixteen heads, pages longer than most sequences, many sequences of one row each."""
    from respect_b200.kernels import paged_attention
    for H, HK, ps, lens in ((70, 2, 1000, [1700, 3, 999, 1001]), (17, 1, 48, [49, 0, 400])):
        q, k, v, table, seqs = paged_inputs(60 + H, lens, H, HK, ps, dtype)
        close(paged_attention(q, k, v, table, i32(lens)), *paged_reference(q, seqs))
    lens = [i % 40 for i in range(700)]
    q, k, v, table, seqs = paged_inputs(63, lens, 4, 1, 16, dtype)
    y = paged_attention(q, k, v, table, i32(lens))
    for b in (0, 1, 39, 355, 699):
        o, t = paged_reference(q[b:b + 1], seqs[b:b + 1])
        close(y[b:b + 1], o, t)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_token_logprobs_many_rows_and_past_32_bits(dtype):
    """More rows than a grid's second dimension could hold, and logits whose elements lie beyond 2^31: the
    bits of the same rows alone."""
    from respect_b200.decoding.acceptance import token_logprobs
    g = gen(64)
    for rows, V, top in ((70000, 50, 3), (15000, 152064, 5)):
        x = torch.empty(rows, V, device=DEV, dtype=dtype)
        for r in range(0, rows, 4096):
            x[r:r + 4096] = randn(g, *x[r:r + 4096].shape, dtype=dtype, scale=3.0)
        tokens = torch.randint(0, V, (rows,), device=DEV, generator=g)
        r = token_logprobs(x, tokens, top, 7, 20)
        some = [0, 1, rows // 2, rows - 2, rows - 1]
        one = token_logprobs(x[some], tokens[some], top, 7, 20)
        tokens_out = (tokens[some] >= 7) & (tokens[some] < 27)      # -inf: equal, too
        assert all(torch.equal(a[some], b) for a, b in zip(r, one)) and bool((r.logprob[some].isinf() == tokens_out).all())
        base.assert_logprobs(x[some], tokens[some], top, 7, 20)
        del x, r


@pytest.mark.parametrize("dtype", [BF, F32])
def test_token_logprobs_masked_by_the_lowest_value(dtype):
    """Entries at the type's lowest value weigh what entries at -inf weigh; a row of nothing else is uniform."""
    from respect_b200.decoding.acceptance import token_logprobs
    V = 30001
    g = gen(65)
    x = randn(g, 4, V, dtype=dtype, scale=3.0)
    tokens = torch.tensor([5, 20000, 17, 3], device=DEV)
    masked = torch.rand(4, V, device=DEV, generator=g) < 0.7
    masked[1, 8192:16384] = True
    masked[torch.arange(4), tokens] = False
    low = x.masked_fill(masked, torch.finfo(dtype).min)
    a, b = token_logprobs(low, tokens, 20), token_logprobs(x.masked_fill(masked, -INF), tokens, 20)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    r = token_logprobs(torch.full_like(x, torch.finfo(dtype).min), tokens, 4)
    want = torch.full((4,), float(V), device=DEV).log()
    # log S of V ones: S good to 2^-17 (see assert_logprobs), and the logarithm's own rounding
    assert bool(((r.logprob + want).abs() <= 2.0 ** -17).all()) and bool(((r.entropy - want).abs() <= 2.0 ** -17).all())
    assert r.top_ids.tolist() == [[0, 1, 2, 3]] * 4


# ---------------------------------------------------------------- calls that nothing above makes
@pytest.mark.parametrize("dtype", [BF, F32])
def test_tables_without_columns_or_rows(dtype):
    from respect_b200.kernels import paged_attention
    q, k, v, table, _ = paged_inputs(66, [30, 5], 8, 2, 16, dtype)
    assert not bool(paged_attention(q, k, v, table[:, :0], i32([30, 5])).any())
    assert not bool(paged_attention(q, k, v, table[:0], i32([]), seqs=i32([0, 1])).any())
    assert not bool(paged_attention(q, k[:0], v[:0], table, i32([30, 5])).any())
    assert not bool(paged_attention(q, k, v, table, i32([0, -7]), ahead=0).any())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_two_streams_at_once_and_a_captured_call_with_bad_values(dtype):
    """The same operators on two streams at a time, and a graph whose replay meets values that are not finite."""
    from respect_b200.decoding.acceptance import token_logprobs
    from respect_b200.kernels import paged_attention, prompt_attention
    q, k, v, cu = prompt_inputs(67, [900, 300], 8, 2, dtype)
    v, cu = v.clone(), i32(cu)
    pq, pk, pv, table, _ = paged_inputs(68, [3000, 700], 8, 2, 16, dtype)
    n = i32([3000, 700])
    x, tok = randn(gen(69), 40, 30000, dtype=dtype), torch.arange(40, device=DEV)

    def everything():
        return (prompt_attention(q, k, v, cu), paged_attention(pq, pk, pv, table, n), *token_logprobs(x, tok, 7))

    want = everything()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(everything())
    torch.cuda.synchronize()
    for y in got:
        assert all(torch.equal(a, b) for a, b in zip(y, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = prompt_attention(q, k, v, cu)
    for token, value in ((890, NAN), (5, INF), (1000, -INF)):
        v[token, 1, 17] = value
        graph.replay()
        again = prompt_attention(q, k, v, cu)
        assert torch.equal(y.nan_to_num(7.0), again.nan_to_num(7.0)) and torch.equal(y.isnan(), again.isnan())
        assert not torch.equal(y[token:token + 1], want[0][token:token + 1])
