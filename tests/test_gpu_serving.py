"""The serving operators on the GPU against plain 64-bit restatements (tests/serving_reference.py, which
derives the tolerances), at the sizes, masks and layouts where they can go wrong."""
import random

import pytest
import torch

from tests.serving_reference import Pages, attention, close

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
SCALE = 128 ** -0.5


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- prompts
def prompt_inputs(seed, lens, H, HK, dtype, before=0, behind=0, scale=1.0):
    T = before + sum(lens) + behind
    qkv = randn(gen(seed), T, H + 2 * HK, 128, dtype=dtype, scale=scale)
    cu = [before]
    for n in lens:
        cu.append(cu[-1] + n)
    return qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:], cu


def prompt_reference(q, k, v, cu, scale=SCALE):
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    weight = 2.0 ** -8 if q.dtype == BF else 0.0
    for a, b in zip(cu, cu[1:]):
        if b > a:
            mask = torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).tril()
            for r in range(0, b - a, 512):
                e = min(b - a, r + 512)
                out[a + r:a + e], tol[a + r:a + e] = attention(q[a + r:a + e], k[a:a + e], v[a:a + e], mask[r:e, :e],
                                                               scale, weight)
    return out, tol


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,HK,lens", [
    (28, 4, [1]), (28, 4, [0, 1, 2, 0]), (28, 4, [37, 0, 19, 128, 5]), (32, 8, [127, 128, 129]), (8, 8, [65, 300]),
    (4, 2, [513]), (40, 8, [1, 257, 31]), (64, 1, [40, 3]), (16, 16, [1, 1, 1, 1]), (6, 2, [1100]),
    (28, 4, list(range(40)))])
def test_prompt_attention(dtype, H, HK, lens):
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(H * 100 + len(lens), lens, H, HK, dtype)
    close(prompt_attention(q, k, v, i32(cu)), *prompt_reference(q, k, v, cu))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_long_and_sharp(dtype):
    """A longer prompt, and scores spread over hundreds (one key takes nearly everything)."""
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(3, [2500], 4, 1, dtype)
    close(prompt_attention(q, k, v, i32(cu)), *prompt_reference(q, k, v, cu))
    # the score error bound grows with the scores: stay where its first order holds
    q, k, v, cu = prompt_inputs(4, [400, 77], 4, 2, dtype, scale=2.0)
    close(prompt_attention(q, k, v, i32(cu), sm_scale=0.5), *prompt_reference(q, k, v, cu, 0.5))
    close(prompt_attention(q, k, v, i32(cu), sm_scale=-0.25), *prompt_reference(q, k, v, cu, -0.25))
    close(prompt_attention(q, k, v, i32(cu), sm_scale=0.0), *prompt_reference(q, k, v, cu, 0.0))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_rows_of_no_sequence_and_given_out(dtype):
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(5, [70, 9], 8, 2, dtype, before=11, behind=23)
    for t in (q, k, v):                       # nobody's rows hold anything at all
        t[:11], t[-23:] = float("nan"), float("inf")
    ref, tol = prompt_reference(q, k, v, cu)
    y = prompt_attention(q, k, v, i32(cu))
    close(y, ref, tol)                        # zeros outside the sequences
    wide = torch.full((q.shape[0], 8, 256), 7.0, device=DEV, dtype=dtype)
    out = wide[:, :, 128:]
    assert prompt_attention(q, k, v, i32(cu), out=out) is out
    assert torch.equal(out[11:-23], y[11:-23])
    assert bool((out[:11] == 7).all()) and bool((out[-23:] == 7).all()) and bool((wide[:, :, :128] == 7).all())
    assert not bool(prompt_attention(q, k, v, i32([0])).any())                 # no sequences
    assert prompt_attention(q[:0], k[:0], v[:0], i32([0, 0])).shape == (0, 8, 128)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_packing_changes_no_bit(dtype):
    from respect_b200.kernels import prompt_attention
    lens = [300, 1, 45, 129]
    q, k, v, cu = prompt_inputs(6, lens, 28, 4, dtype)
    y = prompt_attention(q, k, v, i32(cu))
    for a, b in zip(cu, cu[1:]):
        assert torch.equal(prompt_attention(q[a:b], k[a:b], v[a:b], i32([0, b - a])), y[a:b])
    n = 190                                   # a prompt cut short gives the same rows
    assert torch.equal(prompt_attention(q[:n], k[:n], v[:n], i32([0, n])), y[:n])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_nothing_of_masked_places_shows(dtype, bad):
    """NaN and infinities in later tokens of the same prompt and in other prompts reach no earlier row."""
    from respect_b200.kernels import prompt_attention
    q, k, v, cu = prompt_inputs(7, [150, 40], 4, 2, dtype)
    ref, tol = prompt_reference(q, k, v, cu)
    k2, v2 = k.clone(), v.clone()
    k2[150:], v2[150:] = bad, bad
    k2[101:150], v2[101:150] = bad, bad
    y = prompt_attention(q, k2, v2, i32(cu))
    close(y[:101], ref[:101], tol[:101])
    v3 = v.clone()
    v3[60, 1, 5] = bad                        # one value: only its dim, from its token on
    y = prompt_attention(q, k, v3, i32(cu))
    ref3, tol3 = ref.clone(), tol.clone()
    ref3[60:150, 2:, 5] = bad
    close(y, ref3, tol3)


# ---------------------------------------------------------------- pages
def paged_inputs(seed, lens, H, HK, ps, dtype, spare=3, layout="heads"):
    """Random pages in random order; whatever no sequence holds is NaN."""
    g = gen(seed)
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + spare
    shape = (pages, HK, ps, 128) if layout == "heads" else (pages, ps, HK, 128)
    kv = [torch.full(shape, float("nan"), device=DEV, dtype=dtype) for _ in range(2)]
    if layout != "heads":
        kv = [x.transpose(1, 2) for x in kv]
    order = torch.randperm(pages, device=DEV, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1]) + 2), -1, dtype=torch.int32)
    seqs = []
    for i, n in enumerate(lens):
        kk, vv = randn(g, n, HK, 128, dtype=dtype), randn(g, n, HK, 128, dtype=dtype)
        for j in range(need[i]):
            p = order.pop()
            table[i, j] = p
            m = min(ps, n - j * ps)
            kv[0][p, :, :m] = kk[j * ps:j * ps + m].transpose(0, 1)
            kv[1][p, :, :m] = vv[j * ps:j * ps + m].transpose(0, 1)
        seqs.append((kk, vv))
    return randn(g, len(lens), H, 128, dtype=dtype), kv[0], kv[1], table.to(DEV), seqs


def paged_reference(q, seqs, scale=SCALE, keep=None):
    out, tol = torch.zeros(2, *q.shape, dtype=torch.float64, device=DEV).unbind(0)
    for b, (k, v) in enumerate(seqs):
        mask = torch.ones(1, k.shape[0], dtype=torch.bool, device=DEV)
        if keep is not None:
            mask[0] = keep[b]
        o, t = attention(q[b:b + 1], k, v, mask, scale, 2.0 ** -16 if q.dtype == BF else 0.0)
        out[b], tol[b] = o[0], t[0]
    return out, tol


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,HK,ps,lens", [
    (28, 4, 16, [1, 0, 17, 16, 300]), (32, 8, 64, [1000, 63, 64, 65]), (8, 1, 8, [129, 2]), (16, 16, 24, [50, 128, 127]),
    (40, 2, 100, [777, 5]), (4, 2, 1, [33]), (34, 2, 7, [260]), (28, 4, 128, [9000, 8192, 8193, 0, 1]), (64, 1, 32, [400])])
def test_paged_attention(dtype, H, HK, ps, lens):
    from respect_b200.kernels import paged_attention
    for layout in ("heads", "slots"):
        q, k, v, table, seqs = paged_inputs(H + ps, lens, H, HK, ps, dtype, layout=layout)
        close(paged_attention(q, k, v, table, i32(lens)), *paged_reference(q, seqs))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_paged_rows_lengths_and_out(dtype):
    """Rows picked by seqs (one twice, some outside the table), tokens ahead of the length, bounds on the
    length, strided queries and results."""
    from respect_b200.kernels import paged_attention
    lens = [70, 0, 513, 40]
    q, k, v, table, seqs = paged_inputs(9, lens, 8, 2, 16, dtype)
    ref, tol = paged_reference(q, seqs)
    pick = [2, 0, 2, -1, 4, 3]
    big = torch.zeros(6, 3, 8, 128, device=DEV, dtype=dtype)
    big[:, 1] = torch.stack([q[i] if 0 <= i < 4 else q[0] for i in pick])
    y = paged_attention(big[:, 1], k, v, table, i32(lens), seqs=i32(pick))
    for row, i in enumerate(pick):
        if 0 <= i < 4:
            close(y[row], ref[i], tol[i])
        else:
            assert not bool(y[row].any())
    short = i32([60, 0, 500, 39])
    want, tol2 = paged_reference(q, [(a[:n], b[:n]) for (a, b), n in zip(seqs, [61, 1, 501, 40])])
    t1 = table.clone()
    t1[1, 0] = -1                              # the token ahead of an empty sequence has no page
    want[1], tol2[1] = 0, 0
    close(paged_attention(q, k, v, t1, short, ahead=1), want, tol2)
    for bound in (1, 33, 512):
        want, tol2 = paged_reference(q, [(a[:bound], b[:bound]) for a, b in seqs])
        close(paged_attention(q, k, v, table, i32(lens), max_length=bound), want, tol2)
    # lengths beyond the table and below zero
    want, tol2 = paged_reference(q, seqs)
    full = paged_attention(q, k, v, table[:, :33], i32([70, -5, 1 << 30, 40]))
    want2, tol3 = paged_reference(q, [(a[:528], b[:528]) for a, b in seqs])
    close(full[[0, 1, 3]], want[[0, 1, 3]], tol2[[0, 1, 3]])
    out = torch.full((4, 16, 128), 5.0, device=DEV, dtype=dtype)
    paged_attention(q, k, v, table, i32(lens), out=out[:, 8:])
    close(out[:, 8:], ref, tol)
    assert bool((out[:, :8] == 5).all())
    assert paged_attention(q[:0], k, v, table[:0], i32([])).shape == (0, 8, 128)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_paged_entries_that_name_no_page(dtype):
    from respect_b200.kernels import paged_attention
    lens = [300, 40, 16]
    q, k, v, table, seqs = paged_inputs(11, lens, 28, 4, 16, dtype)
    table[0, 3], table[0, 18], table[2, 0] = -1, k.shape[0], 1 << 30
    keep = [torch.ones(n, dtype=torch.bool, device=DEV) for n in lens]
    keep[0][48:64], keep[0][288:300], keep[2][:] = False, False, False
    close(paged_attention(q, k, v, table, i32(lens)), *paged_reference(q, seqs, keep=keep))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_paged_batch_changes_no_bit_and_values_travel(dtype):
    from respect_b200.kernels import paged_attention
    lens = [300, 4500, 1, 128, 129]
    q, k, v, table, seqs = paged_inputs(12, lens, 28, 4, 16, dtype)
    y = paged_attention(q, k, v, table, i32(lens))
    for b in range(5):
        assert torch.equal(paged_attention(q[b:b + 1], k, v, table, i32(lens), seqs=i32([b])), y[b:b + 1])
    # an infinity or NaN that is attended shows where it belongs
    page, slot = int(table[0, 5]), 3
    for bad in (float("inf"), float("-inf"), float("nan")):
        v2 = v.clone()
        v2[page, 1, slot, 9] = bad
        ref, tol = paged_reference(q, seqs)
        ref[0, 7:14, 9] = bad
        close(paged_attention(q, k, v2, table, i32(lens)), ref, tol)


def test_paged_offsets_past_32_bits():
    """Pages that lie more than 2^31 elements into the cache."""
    from respect_b200.kernels import paged_attention
    pages, HK, ps = 70000, 4, 64
    k = torch.empty(pages, HK, ps, 128, device=DEV, dtype=BF)      # 2.3e9 elements
    g = gen(13)
    rows = [pages - 1, 3, pages - 20]
    kk = randn(g, 150, HK, 128, dtype=BF)
    for j, p in enumerate(rows):
        m = min(ps, 150 - j * ps)
        k[p, :, :m] = kk[j * ps:j * ps + m].transpose(0, 1)
    q = randn(g, 1, 28, 128, dtype=BF)
    close(paged_attention(q, k, k, i32([rows]), i32([150])), *paged_reference(q, [(kk, kk)]))


def test_captured_and_on_another_stream():
    """Calls captured into two graphs, replayed on new inputs; eager calls on a side stream."""
    from respect_b200.decoding.acceptance import token_logprobs
    from respect_b200.kernels import paged_attention, prompt_attention
    lens = [700, 33]
    q, k, v, table, _ = paged_inputs(14, lens, 8, 2, 16, BF)
    n = i32(lens)
    pq, pk, pv, cu = prompt_inputs(15, [90, 41], 8, 2, BF)
    pq, pk, pv, cu = pq.clone(), pk.clone(), pv.clone(), i32(cu)
    x, tok = randn(gen(16), 3, 20000), torch.tensor([5, 19999, 7], device=DEV)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (paged_attention(q, k, v, table, n), prompt_attention(pq, pk, pv, cu), *token_logprobs(x, tok, 4))
        graphs.append((graph, out))
    for seed in (17, 18):
        q.copy_(randn(gen(seed), *q.shape, dtype=BF))
        pq.copy_(randn(gen(seed + 9), *pq.shape, dtype=BF))
        x.copy_(randn(gen(seed + 3), *x.shape))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = (paged_attention(q, k, v, table, n), prompt_attention(pq, pk, pv, cu), *token_logprobs(x, tok, 4))
        torch.cuda.current_stream().wait_stream(side)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_expanded_and_turned_inputs():
    """Inputs whose rows repeat in place or lie the other way round are read as what they are."""
    from respect_b200.decoding.acceptance import token_logprobs
    from respect_b200.decoding.kv_pages import PagedKVCache
    from respect_b200.kernels import paged_attention, prompt_attention
    g = gen(40)
    for dtype in (BF, F32):
        q, k, v, table, seqs = paged_inputs(41, [70], 8, 2, 16, dtype)
        q3 = randn(g, 3, 8, 128, dtype=dtype)
        want, tol = paged_reference(q3, seqs * 3)
        close(paged_attention(q3, k, v, table.expand(3, -1), i32([70]).expand(3)), want, tol)
        close(paged_attention(q3, k, v, table.t().contiguous().t().expand(3, -1), i32([70, 70, 70])), want, tol)
        kv1 = k[:, :1].expand(-1, 2, -1, -1)             # one head read as two
        close(paged_attention(q3, kv1, kv1, table.expand(3, -1), i32([70] * 3)),
              *paged_reference(q3, [(seqs[0][0][:, :1].expand(-1, 2, -1),) * 2] * 3))
        pq, pk, pv, cu = prompt_inputs(42, [50, 33], 8, 2, dtype)
        one = pk[:, :1].expand(-1, 2, -1)
        close(prompt_attention(pq, one, one, i32(cu)), *prompt_reference(pq, one, one, cu))
        turned = pq.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(prompt_attention(turned, pk, pv, i32(cu)), prompt_attention(pq, pk, pv, i32(cu)))
        odd = randn(g, 83, 8, 129, dtype=dtype)[:, :, 1:]   # rows off the 16-byte grid
        close(prompt_attention(odd, pk, pv, i32(cu)), *prompt_reference(odd, pk, pv, cu))
    x = randn(g, 1, 9000).expand(4, -1)
    tok = torch.tensor([3, 3, 5, 5], device=DEV)
    a = token_logprobs(x, tok, 5)
    b = token_logprobs(x.contiguous(), tok, 5)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    cache = PagedKVCache(1, 1, 16, 4, 3, dtype=F32)
    cache.reserve([0, 1, 2], [6, 6, 6])
    cache.write(*token_kv(cache, list(range(18))), [0, 1, 2], [0, 6, 12, 18])
    cache.compact([0, 1, 2], i32([[1, 4]]).expand(3, -1), i32([2]).expand(3))
    cache.check()
    assert cache.lengths.tolist() == [2, 2, 2] and cache.held.tolist() == [1, 1, 1]
    for s, want in enumerate(([1, 4], [7, 10], [13, 16])):
        k, _ = token_kv(cache, want)
        assert torch.equal(cache.store[0, 0, cache.table[s, 0], 0, :2], k[0, :, 0])


def test_reserve_of_more_than_32_bits_can_count():
    """Many sequences asking for everything: refused, nothing changed."""
    from respect_b200.decoding.kv_pages import PagedCacheError, PagedKVCache
    cache = PagedKVCache(1, 1, 4, 1, 1000, max_pages=3_000_000, head_dim=8)
    cache.reserve(list(range(1000)), [3_000_000] * 1000)
    with pytest.raises(PagedCacheError, match="free pages"):
        cache.check()
    assert not bool(cache.refs.any()) and not bool(cache.held.any())


# ---------------------------------------------------------------- page operations
def token_kv(cache, tokens):
    """K / V [layers, n, heads, D] that encode token numbers: distinct for layer, side and head."""
    L, HK, D = cache.layers, cache.kv_heads, cache.head_dim
    base = torch.tensor(tokens, device=DEV, dtype=F32).reshape(1, -1, 1, 1) * 4
    part = torch.arange(L * HK, device=DEV, dtype=F32).reshape(L, 1, HK, 1) / 64
    k = (base + part + torch.arange(D, device=DEV) / 4096).to(cache.dtype)
    return k, -k


def assert_same(cache, model):
    assert cache.lengths.tolist() == model.lengths
    assert cache.held.tolist() == [len(r) for r in model.rows]
    assert cache.refs.tolist() == model.refs
    for i, r in enumerate(cache.table.tolist()):
        assert r[:len(model.rows[i])] == model.rows[i] and all(x == -1 for x in r[len(model.rows[i]):])
    for s in range(len(model.rows)):
        tokens = model.tokens(s)
        if not tokens:
            continue
        pos = torch.arange(len(tokens), device=DEV)
        page, slot = cache.table[s].long()[pos // cache.page_size], pos % cache.page_size
        k, v = token_kv(cache, tokens)
        assert torch.equal(cache.store[:, 0][:, page, :, slot].transpose(0, 1), k)
        assert torch.equal(cache.store[:, 1][:, page, :, slot].transpose(0, 1), v)


@pytest.mark.parametrize("ps,pages,dtype,layers,heads,dim", [
    (4, 40, F32, 2, 2, 128), (16, 30, F32, 1, 3, 128), (1, 120, F32, 3, 1, 8), (7, 64, F32, 2, 2, 20)])
def test_page_operations_follow_the_model(ps, pages, dtype, layers, heads, dim):
    """Random sequences of operations against a plain model, token by token; calls the pool cannot
    serve change nothing and say so."""
    from respect_b200.decoding.kv_pages import PagedCacheError, PagedKVCache
    rng = random.Random(ps)
    N = 6
    cache = PagedKVCache(layers, heads, pages, ps, N, max_pages=24, head_dim=dim, dtype=dtype)
    model = Pages(pages, ps, N, 24)
    token, refused = 1, 0
    for step in range(120):
        op = rng.choice(["grow", "grow", "round", "fork", "truncate", "free"])
        seqs = rng.sample(range(N), rng.randint(1, N))
        if op in ("grow", "round"):
            counts = [rng.randint(0, min(2 * ps + 3, 24 * ps - model.lengths[s])) for s in seqs]
            cache.reserve(seqs, counts)
            if not model.reserve(seqs, counts):
                refused += 1
                with pytest.raises(PagedCacheError, match="free pages"):
                    cache.check()
                assert_same(cache, model)
                drop = rng.randrange(N)
                cache.free([drop])
                model.truncate(drop, 0)
                continue
            news = [list(range(token + sum(counts[:i]), token + sum(counts[:i + 1]))) for i in range(len(seqs))]
            token += sum(counts)
            k, v = token_kv(cache, [t for x in news for t in x])
            offsets = [0]
            for c in counts:
                offsets.append(offsets[-1] + c)
            if rng.random() < 0.5:
                cache.write(k, v, seqs, offsets)
            else:
                for layer in range(layers):
                    cache.write(k[layer], v[layer], seqs, i32(offsets), layer=layer)
            for s, x in zip(seqs, news):
                model.write(s, x)
            if op == "grow":
                cache.commit(seqs, i32(counts))
                for s, c in zip(seqs, counts):
                    model.commit(s, c)
            else:
                paths = [sorted(rng.sample(range(c), rng.randint(0, c))) for c in counts]
                cache.compact(seqs, paths, [len(x) for x in paths])
                for s, x in zip(seqs, paths):
                    model.compact(s, x)
        elif op == "fork":
            empty = [s for s in range(N) if not model.rows[s]]
            full = [s for s in range(N) if model.rows[s]]
            if not empty or not full:
                continue
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(full) for _ in dst]
            cache.fork(src, dst)
            for a, d in zip(src, dst):
                model.fork(a, d)
        elif op == "truncate":
            keep = [rng.randint(0, model.lengths[s]) for s in seqs]
            cache.truncate(seqs, keep)
            for s, n in zip(seqs, keep):
                model.truncate(s, n)
        else:
            cache.free(seqs[:2])
            for s in seqs[:2]:
                model.truncate(s, 0)
        cache.check()
        if step % 6 == 0:
            assert_same(cache, model)
    assert_same(cache, model)


def test_page_operations_refuse_and_change_nothing():
    from respect_b200.decoding.kv_pages import PagedCacheError, PagedKVCache
    cache = PagedKVCache(2, 2, 12, 4, 4, max_pages=8)
    cache.reserve([0, 1], [6, 3])
    k, v = token_kv(cache, list(range(9)))
    cache.write(k, v, [0, 1], [0, 6, 9])
    cache.commit([0, 1], [6, 3])
    cache.check()

    def same(what, match):
        before = [t.clone() for t in (cache.store, cache.table, cache.lengths, cache.held, cache.refs)]
        what()
        with pytest.raises(PagedCacheError, match=match):
            cache.check()
        cache.check()       # cleared
        for a, b in zip(before, (cache.store, cache.table, cache.lengths, cache.held, cache.refs)):
            assert torch.equal(a, b)

    named = "named twice"
    room = "room"
    for bad in ([0, 0], [0, 4], [-1, 0]):
        same(lambda: cache.reserve(bad, [1, 1]), named)
        same(lambda: cache.commit(bad, [0, 0]), named)
        same(lambda: cache.truncate(bad, [0, 0]), named)
        same(lambda: cache.free(bad), named)
        same(lambda: cache.compact(bad, [[], []], [0, 0]), named)
    for src, dst in (([0, 0], [2, 2]), ([0], [1]), ([0], [0]), ([4], [2]), ([0, 2], [2, 3]), ([0], [9])):
        same(lambda: cache.fork(src, dst), named)
    same(lambda: cache.reserve([0, 2], [1, 100]), room)            # past the table's width
    same(lambda: cache.reserve([0], [-1]), room)
    same(lambda: cache.reserve([0, 1, 2, 3], [26, 29, 20, 20]), "free pages")
    same(lambda: cache.commit([1, 0], [0, 3]), room)               # 9 tokens in two pages
    same(lambda: cache.commit([0], [-1]), room)
    same(lambda: cache.truncate([1, 0], [1, 7]), room)
    same(lambda: cache.truncate([0], [-1]), room)
    same(lambda: cache.compact([0], [[0, 2]], [2]), room)          # room for two more tokens only
    same(lambda: cache.compact([0], [[1, 1]], [2]), room)
    same(lambda: cache.compact([0], [[1, 0]], [2]), room)
    same(lambda: cache.compact([0], [[-1]], [1]), room)
    same(lambda: cache.compact([0], [[0]], [2]), room)
    one = token_kv(cache, [77])
    same(lambda: cache.write(*one, [2]), room)                     # nothing reserved
    same(lambda: cache.write(*token_kv(cache, [1, 2]), [0, 0]), named)
    same(lambda: cache.write(*one, [-3]), named)
    cache.fork([0], [2])
    same(lambda: cache.write(*one, [0]), "another sequence holds")
    same(lambda: cache.compact([0], [[0]], [1]), "another sequence holds")
    # tokens of nobody are left out without a word
    cache.write(*token_kv(cache, [50, 51, 52]), [1], [3, 3])
    cache.check()
    # empty lists
    cache.reserve([], [])
    cache.commit([], [])
    cache.fork([], [])
    cache.free([])
    cache.compact([], [], [])
    cache.check()


def test_counts_beyond_the_table():
    """A state whose counts name more than a row of the table holds: the next rows stay as they were."""
    from respect_b200.decoding.kv_pages import PagedCacheError, PagedKVCache
    cache = PagedKVCache(1, 1, 32, 4, 4, max_pages=4, dtype=F32)
    cache.reserve([0, 1], [16, 16])
    cache.commit([0, 1], [16, 16])
    cache.held[0], cache.lengths[0] = 8, 32
    cache.reserve([0], [1])                 # its row is full
    with pytest.raises(PagedCacheError, match="room"):
        cache.check()
    cache.fork([0], [2])
    cache.check()
    assert cache.lengths[2].item() == 16 and torch.equal(cache.table[2], cache.table[0])
    cache.free([0])
    cache.check()
    assert cache.table[0].tolist() == [-1] * 4 and cache.table[1].tolist() == [4, 5, 6, 7]
    assert cache.refs.tolist() == [1] * 8 + [0] * 24
    assert cache.held.tolist() == [0, 4, 4, 0] and cache.lengths.tolist() == [0, 16, 16, 0]
    cache.held[3], cache.lengths[3] = -2, -9
    cache.reserve([3], [5])
    cache.check()
    assert cache.held[3].item() == 2 and cache.table[3].tolist() == [8, 9, -1, -1]


def test_forks_of_long_tables():
    """Tables too large for the plan's own block: the same result through a block per pair."""
    from respect_b200.decoding.kv_pages import PagedKVCache
    cache = PagedKVCache(1, 1, 3000, 2, 8, max_pages=5000, dtype=F32)
    model = Pages(3000, 2, 8, 5000)
    cache.reserve([1, 6], [4001, 333])
    cache.commit([1, 6], [4001, 333])
    cache.fork([1, 6, 1, 6], [0, 7, 3, 2])
    cache.check()
    model.reserve([1, 6], [4001, 333])
    model.lengths[1], model.lengths[6] = 4001, 333
    for a, d in ((1, 0), (6, 7), (1, 3), (6, 2)):
        model.fork(a, d)
    assert cache.lengths.tolist() == model.lengths and cache.refs.tolist() == model.refs
    assert cache.held.tolist() == [len(r) for r in model.rows]
    for i, r in enumerate(cache.table.tolist()):
        assert [x for x in r if x >= 0] == model.rows[i]


def test_page_operations_captured():
    """A decoding round captured once and replayed: each replay is the next token."""
    from respect_b200.decoding.kv_pages import PagedKVCache
    cache = PagedKVCache(2, 2, 16, 4, 3, dtype=F32)
    model = Pages(16, 4, 3, 16)
    seqs, ones = i32([0, 2]), i32([1, 1])
    k, v = (t.clone() for t in token_kv(cache, [0, 0]))
    q = randn(gen(20), 2, 4, 128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reserve(seqs, ones)
        cache.write(k, v, seqs)
        y = cache.attend(q, seqs, 1, ahead=1)
        cache.commit(seqs, ones)
    for step in range(9):
        new = [10 + 2 * step, 11 + 2 * step]
        for dst, src in zip((k, v), token_kv(cache, new)):
            dst.copy_(src)
        graph.replay()
        model.reserve([0, 2], [1, 1])
        for s, t in zip([0, 2], new):
            model.write(s, [t])
            model.commit(s, 1)
        assert_same(cache, model)
        want = [token_kv(cache, model.tokens(s)) for s in (0, 2)]
        close(y, *paged_reference(q, [(a[1], b[1]) for a, b in want]))
    cache.check()


# ---------------------------------------------------------------- log probabilities
def logprob_reference(x, tokens, top, off, size):
    x = x.double().clone()
    x[:, off:off + size] = float("-inf")
    lp = torch.log_softmax(x, 1)
    bad = x.isnan().any(1) | (x == float("inf")).any(1) | (x == float("-inf")).all(1)
    lp[bad] = float("nan")
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    ent[bad] = float("nan")
    ok = (tokens >= 0) & (tokens < x.shape[1])
    at = torch.where(ok, lp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0], float("nan"))
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return at, ent, lp.gather(1, ids), ids


def assert_logprobs(x, tokens, top, off=0, size=0):
    """fp32 results: log p = x - m - log S. S sums V exponentials, each good to 2^-22 and a rounding of its
    argument (2^-24 |x - m| log2 e, small where it counts), in sums that chain fewer than 64 + V / 8192
    roundings: S is good to 2^-21 + (64 + V / 8192) 2^-24 < 2^-17 for V <= 2^19, and so is log S absolutely; the two
    differences round by 2^-24 of |x|, |m| and the result."""
    from respect_b200.decoding.acceptance import token_logprobs
    r = token_logprobs(x, tokens, top, off, size)
    at, ent, lps, ids = logprob_reference(x, tokens, top, off, size)
    big = x.double().masked_fill(~x.isfinite(), 0.0).abs().amax(1)
    s = 2.0 ** -17 + 2.0 ** -22 * (big + 20)

    def near(got, ref, tol):
        same = (got.double() == ref) | (got.isnan() & ref.isnan())
        assert bool((same | ((got.double() - ref).abs() <= tol)).all()), (got.double() - ref).abs().max()
    near(r.logprob, at, s + 2.0 ** -23 * at.nan_to_num(0, 0, 0).abs())
    # H = log S - T / S; T's terms d e^d are good like S's, and |T| <= S (log V + 1)
    near(r.entropy, ent, s * (2 + ent.nan_to_num(0).abs()))
    if top:
        assert torch.equal(r.top_ids, ids)
        near(r.top_logprobs, lps, s[:, None] + 2.0 ** -23 * lps.nan_to_num(0, 0, 0).abs())
    else:
        assert r.top_ids is None and r.top_logprobs is None


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,V,top", [(1, 152064, 20), (3, 8192, 32), (5, 8193, 5), (2, 40, 32), (7, 33, 0), (1, 1, 1),
                                        (4, 32000, 1), (130, 2049, 7), (2, 24601, 32)])
def test_token_logprobs(dtype, rows, V, top):
    g = gen(rows + V)
    x = randn(g, rows, V, dtype=dtype, scale=4.0)      # bf16 values tie often
    assert_logprobs(x, torch.randint(0, V, (rows,), device=DEV, generator=g), top)
    off, size = V // 3, V // 4
    assert_logprobs(x, torch.randint(0, V, (rows,), device=DEV, generator=g), top, off, size)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_token_logprobs_hard_rows(dtype):
    """Ties everywhere, huge and tiny values, signed zeros, infinities, NaN, everything excluded."""
    V = 20000
    g = gen(21)
    x = randn(g, 10, V, dtype=dtype)
    x[0] = 0.0
    x[1] = torch.where(torch.arange(V, device=DEV) % 2 == 0, -0.0, 0.0)
    x[2] = float("-inf")
    x[3, 17] = float("inf")
    x[4, 9000] = float("nan")
    x[5] = float("-inf")
    x[5, 12345] = 3.0
    x[6] = x[6] * 1e4
    x[7] = x[7] + 300.0
    x[8, 8190:8200] = 50.0
    x[9] = torch.linspace(-60, 60, V, device=DEV)       # a thread's entries are all among the best
    tokens = torch.tensor([0, V - 1, 3, 17, 2, 12345, -1, V, 8195, V - 1], device=DEV)
    assert_logprobs(x, tokens, 32)
    assert_logprobs(x, tokens, 5, 8000, 12000)
    assert_logprobs(x, tokens, 3, 0, V)                 # nothing left
    assert_logprobs(x, tokens, 32, 20, V)               # fewer entries than alternatives: excluded ones follow


@pytest.mark.parametrize("dtype", [F32, BF])
def test_token_logprobs_layouts(dtype):
    """Rows at every alignment give the bits of an aligned copy; leading dims; strides; one row among many."""
    from respect_b200.decoding.acceptance import greedy_token, token_logprobs
    V = 9001
    g = gen(22)
    big = randn(g, 6, V + 9, dtype=dtype, scale=3.0)
    tokens = torch.randint(0, V, (6,), device=DEV, generator=g)
    for at in (0, 1, 3, 4, 8):
        view = big[:, at:at + V]
        a, b = token_logprobs(view, tokens, 6, 100, 50), token_logprobs(view.clone(), tokens, 6, 100, 50)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        one = token_logprobs(view[4:5], tokens[4:5], 6, 100, 50)
        assert all(torch.equal(x[4:5], y) for x, y in zip(a, one))
        assert torch.equal(a.top_ids[:, 0], greedy_token(view.contiguous(), 100, 50))
    cube = big[:, :V].reshape(2, 3, V)
    r = token_logprobs(cube, tokens.reshape(2, 3), 4)
    assert r.logprob.shape == (2, 3) and r.top_ids.shape == (2, 3, 4)
    assert torch.equal(r.top_ids.reshape(6, 4), token_logprobs(big[:, :V], tokens, 4).top_ids)
    turned = big[:, :V].t().contiguous().t()
    assert torch.equal(token_logprobs(turned, tokens).logprob, token_logprobs(big[:, :V], tokens).logprob)
    assert token_logprobs(big[:0, :V], tokens[:0], 2).top_ids.shape == (0, 2)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_pages_samples_and_logprobs_together(dtype):
    """Two prompts are attended to and cached, samples fork off them and decode token by token, a drafted
    path is compacted; every decoded row equals prompt attention over the sequence's whole text."""
    from respect_b200.decoding.acceptance import token_logprobs
    from respect_b200.decoding.kv_pages import PagedKVCache
    from respect_b200.kernels import prompt_attention
    H, HK, L, V = 8, 2, 2, 500
    g = gen(30)
    cache = PagedKVCache(L, HK, 64, 16, 5, dtype=dtype)
    lens = [37, 150]
    cu = [0, 37, 187]
    qkv = randn(g, L, 187, H + 2 * HK, 128, dtype=dtype)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + HK], qkv[:, :, H + HK:]
    for layer in range(L):
        ref, tol = prompt_reference(q[layer], k[layer], v[layer], cu)
        close(prompt_attention(q[layer], k[layer], v[layer], i32(cu)), ref, tol)
    cache.reserve([0, 1], lens)
    cache.write(k, v, [0, 1], cu)
    cache.commit([0, 1], lens)
    cache.fork([0, 1, 1], [2, 3, 4])
    text = {s: [(k[:, a:b], v[:, a:b])] for s, (a, b) in {2: (0, 37), 3: (37, 187), 4: (37, 187)}.items()}
    seqs = [2, 3, 4]

    def history(s, layer):
        return tuple(torch.cat([x[i][layer] for x in text[s]]) for i in (0, 1))

    for step in range(3):
        new = randn(g, L, 3, H + 2 * HK, 128, dtype=dtype)
        cache.reserve(seqs, [1, 1, 1])
        for i, s in enumerate(seqs):
            text[s].append((new[:, i:i + 1, H:H + HK], new[:, i:i + 1, H + HK:]))
        for layer in range(L):
            cache.write(new[layer, :, H:H + HK], new[layer, :, H + HK:], i32(seqs), layer=layer)
            y = cache.attend(new[layer, :, :H], i32(seqs), layer, ahead=1)
            close(y, *paged_reference(new[layer, :, :H], [history(s, layer) for s in seqs]))
        cache.commit(seqs, [1, 1, 1])
    # a draft of 20 nodes on one sample, of which 3 stay
    draft = randn(g, 2, L, 20, HK, 128, dtype=dtype)
    cache.reserve([3], [20])
    cache.write(draft[0], draft[1], [3], [0, 20])
    cache.compact([3], [[2, 7, 19]], [3])
    text[3].append((draft[0][:, [2, 7, 19]], draft[1][:, [2, 7, 19]]))
    for layer in range(L):
        y = cache.attend(new[layer, :, :H], i32(seqs), layer)
        close(y, *paged_reference(new[layer, :, :H], [history(s, layer) for s in seqs]))
    # the prompts are untouched
    y = cache.attend(q[0, [36, 186]], i32([0, 1]), 0)
    close(y, *paged_reference(q[0, [36, 186]], [(k[0, :37], v[0, :37]), (k[0, 37:], v[0, 37:])]))
    cache.free([0, 1, 2, 3, 4])
    cache.check()
    assert not bool(cache.refs.any()) and bool((cache.table == -1).all())
    x = randn(g, 3, V, scale=3.0)
    assert_logprobs(x, torch.tensor([1, 2, 499], device=DEV), 4)
