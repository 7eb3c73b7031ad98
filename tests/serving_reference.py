"""Plain 64-bit restatements of the serving operators and the tolerances their tests hold them to.

Attention: with weights p (sum 1) and A = sum_j p_j |v_j|, an output o = sum_j p_j v_j is off by at most
  * its one rounding to the output type: eps/2 |o| (bf16 2^-8, fp32 2^-24);
  * the rounding of the weights that enter P V: u A, with u = 2^-8 where one bf16 part carries them
    (bf16 prompts), 2^-16 where two do (bf16 pages), nothing in fp32;
  * the scores' own error ds: every weight changes by a factor within e^(2 ds), so 2 ds A (first order;
    ds <= 0.01 here). A score sums 128 products; with products good to 2^-22 (three tf32 terms) or exact
    (bf16) and an fp32 sum whose partial sums are within S = scale sum_d |q_d k_d|, ds <= (2^-22 + 2^-18) S
    (at most 64 roundings of 2^-24 S are taken one after another);
  * fp32 sums of n weighted values and of n weights: within 64 chained roundings per running sum and a
    rescaling per tile of at least 16 keys, 2 (64 + n / 16) 2^-24 A; the exponential's 2^-22 adds 2^-20 A."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def attention(q, k, v, allowed, scale, weight_error):
    """q [n, H, D], k, v [m, HK, D], allowed bool [n, m] -> (out [n, H, D], tolerance), both fp64; rows that
    attend to nothing are zero."""
    n, H, D = q.shape
    dt = q.dtype
    G = H // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    # what nobody may attend to takes no part, whatever it holds
    used = allowed.any(0)
    k, v, allowed = k[used], v[used], allowed[:, used]
    s = torch.einsum("nhd,mhd->hnm", q, k) * scale
    mag = torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()) * abs(scale)
    s = s.masked_fill(~allowed[None], float("-inf"))
    some = allowed.any(1)
    p = torch.softmax(s[:, some], -1)
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    out[some] = torch.einsum("hnm,mhd->nhd", p, v)
    A = torch.zeros_like(out)
    A[some] = torch.einsum("hnm,mhd->nhd", p, v.abs())
    ds = torch.zeros(n, H, 1, dtype=torch.float64, device=q.device)
    if allowed.numel():
        worst = mag.masked_fill(~allowed[None], 0.0).amax(-1) if k.shape[0] else mag.new_zeros(H, n)
        ds[:, :, 0] = (2.0 ** -22 + 2.0 ** -18) * worst.T
    sums = 2 * (64 + k.shape[0] / 16) * 2.0 ** -24 + 2.0 ** -20
    tol = HALF_STEP[dt] * (out.abs() + weight_error * A) + (weight_error + 2 * ds + sums) * A
    return out, tol


def close(got, ref, tol):
    """got within tol of ref everywhere; NaN and infinities in the same places."""
    got = got.double()
    finite = ref.isfinite()
    assert torch.equal(got.isnan(), ref.isnan()), "NaN in other places"
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), "infinities differ"
    over = ((got - ref).abs() - tol)[finite]
    assert over.numel() == 0 or float(over.max()) <= 0, f"off by {float(over.max()):.3e} more than allowed"


class Pages:
    """A plain model of the paged cache's tables: lists on the host, one token at a time."""

    def __init__(self, pages, page_size, max_seqs, max_pages):
        self.ps, self.max_pages = page_size, max_pages
        self.refs = [0] * pages
        self.rows = [[] for _ in range(max_seqs)]
        self.lengths = [0] * max_seqs
        self.data = {}          # (page, slot) -> token

    def _take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, seqs, counts):
        """False (nothing changed) where the pool runs out."""
        saved = ([list(r) for r in self.rows], list(self.refs), dict(self.data))
        try:
            for s, c in zip(seqs, counts):
                n, row = self.lengths[s], self.rows[s]
                if c and n % self.ps and self.refs[row[n // self.ps]] > 1:
                    old = row[n // self.ps]
                    new = self._take()
                    for i in range(n % self.ps):
                        self.data[new, i] = self.data[old, i]
                    row[n // self.ps] = new
                    self.refs[old] -= 1
                while len(row) * self.ps < n + c:
                    row.append(self._take())
            return True
        except ValueError:
            self.rows, self.refs, self.data = saved
            return False

    def write(self, s, tokens):
        for j, t in enumerate(tokens):
            pos = self.lengths[s] + j
            self.data[self.rows[s][pos // self.ps], pos % self.ps] = t

    def commit(self, s, n):
        self.lengths[s] += n

    def fork(self, a, d):
        n = self.lengths[a]
        self.rows[d] = self.rows[a][:-(-n // self.ps)]
        for p in self.rows[d]:
            self.refs[p] += 1
        self.lengths[d] = n

    def truncate(self, s, n):
        while len(self.rows[s]) > -(-n // self.ps):
            self.refs[self.rows[s].pop()] -= 1
        self.lengths[s] = n

    def compact(self, s, path):
        n = self.lengths[s]
        at = [(self.rows[s][(n + j) // self.ps], (n + j) % self.ps) for j in range((max(path) if path else -1) + 1)]
        for i, a in enumerate(path):
            self.data[at[i]] = self.data[at[a]]
        self.truncate(s, n + len(path))

    def tokens(self, s):
        return [self.data[self.rows[s][i // self.ps], i % self.ps] for i in range(self.lengths[s])]
