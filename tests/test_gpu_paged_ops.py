"""Operators over caller-owned K/V pages against their definitions in 64 bits:
vvq2_attention_paged, vvq2_attention_key_weights, vvq2_pages_evict.

Tolerances are bounds, element by element, from the arithmetic:
* a score is a product of f16 / bf16 values summed in f32 over head_dim terms:
  off by at most hd * 2^-23 * scale * sum |q_i k_i| (each addition rounded or
  cut to 2^-23 relative), E below;
* exp of it, the running rescale factors and the statistics add a few f32
  roundings of |x| <= 2^7 at most: 2^-24 * 2^7 = 2^-17 at the extreme, taken
  relative to every probability;
* the probabilities are rounded to the pages' type before the product with V
  (eps / 2 each, and 2^-25 absolute where f16 probabilities are subnormal),
  the sums over n keys are f32 (n * 2^-23), the output is rounded once
  (eps / 2, and 2^-25 absolute for f16 subnormals)."""
import math

import pytest

import vvq2

pytestmark = pytest.mark.gpu
PAGE = 64
SMALL = 2.0 ** -17


def T():
    import torch
    return torch


def table(lens, rng, n_pages=None, first=0):
    torch = T()
    n = [(l + PAGE - 1) // PAGE for l in lens]
    total = max(1, sum(n)) if n_pages is None else n_pages
    perm = (torch.randperm(total, generator=rng) + first).to(torch.int32)
    bt = torch.full((len(lens), max(1, max(n)) + 1), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(n):
        bt[s, :k] = perm[at:at + k]
        at += k
    return bt, total


class Chunk:
    """Sequences (new tokens, cached keys), their pages (NaN wherever no key
    lives) and packed queries."""

    def __init__(self, seqs, heads, dtype, seed=1, pad=0, qscale=2.0, layers=None, q_extra=0):
        torch = T()
        self.seqs, (self.nq, self.nkv, self.hd) = seqs, heads
        self.G = self.nq // self.nkv
        self.dtype = dtype
        rng = torch.Generator().manual_seed(seed)
        self.bt, pages = table([kv for _, kv in seqs], rng)
        shape = (pages + 1, self.nkv, PAGE, self.hd)
        self.K = torch.full(shape, float("nan"), dtype=dtype)
        self.V = torch.full(shape, float("nan"), dtype=dtype)
        self.keys, self.vals = [], []
        for s, (n, kv) in enumerate(seqs):
            k = torch.randn((kv, self.nkv, self.hd), generator=rng).to(dtype)
            v = torch.randn((kv, self.nkv, self.hd), generator=rng).to(dtype)
            self.keys.append(k)
            self.vals.append(v)
            for p in range((kv + PAGE - 1) // PAGE):
                part = k[p * PAGE:(p + 1) * PAGE]
                self.K[self.bt[s, p], :, :len(part)] = part.transpose(0, 1)
                self.V[self.bt[s, p], :, :len(part)] = v[p * PAGE:(p + 1) * PAGE].transpose(0, 1)
        self.starts = [0]
        for n, _ in seqs:
            self.starts.append(self.starts[-1] + n)
        self.total = self.starts[-1] + pad
        self.q = (torch.randn((self.total, self.nq, self.hd), generator=rng) * qscale).to(dtype)
        self.scale = 1.0 / math.sqrt(self.hd)
        self.max_q = max(1, max(n for n, _ in seqs))
        self.max_kv = max(kv for _, kv in seqs)

    def gpu(self):
        torch = T()
        d = "cuda:0"
        self.pages = vvq2.Pages(self.K.to(d), self.V.to(d), self.bt.to(d))
        self.qd = self.q.to(d)
        self.qs = torch.tensor(self.starts, dtype=torch.int32, device=d)
        self.kl = torch.tensor([kv for _, kv in self.seqs], dtype=torch.int32, device=d)
        return self

    def attend(self, **kw):
        return vvq2.attention_paged(self.qd, self.pages, self.qs, self.kl, self.max_q, self.max_kv, want_lse=True,
                                    **kw)

    def reference(self):
        """out, bound, lse, lse bound (f64, on the GPU) of the packed rows."""
        torch = T()
        d = "cuda:0"
        R = self.starts[-1]
        out = torch.zeros((R, self.nq, self.hd), dtype=torch.float64, device=d)
        tol = torch.zeros_like(out)
        lse = torch.full((R, self.nq), -math.inf, dtype=torch.float64, device=d)
        ltol = torch.zeros_like(lse)
        u = torch.finfo(self.dtype).eps / 2
        for s, (n, kv) in enumerate(self.seqs):
            for g in range(self.nkv):
                K, V = self.keys[s][:, g].to(d).double(), self.vals[s][:, g].to(d).double()
                step = max(1, (1 << 24) // max(1, kv * self.G))
                for t0 in range(0, n, step):
                    t1 = min(n, t0 + step)
                    rows, hs = slice(self.starts[s] + t0, self.starts[s] + t1), slice(g * self.G, (g + 1) * self.G)
                    q = self.q[rows, hs].to(d).double()
                    x = torch.einsum("thd,jd->thj", q, K) * self.scale
                    E = self.hd * 2.0 ** -23 * self.scale * torch.einsum("thd,jd->thj", q.abs(), K.abs())
                    lim = kv - n + torch.arange(t0, t1, device=d) + 1
                    seen = torch.arange(kv, device=d)[None, :] < lim[:, None]
                    x = x.masked_fill(~seen[:, None, :], -math.inf)
                    E = E.masked_fill(~seen[:, None, :], 0).amax(-1) if kv else torch.zeros(x.shape[:2], device=d)
                    some = (lim > 0)[:, None].expand(x.shape[:2])
                    z = torch.where(some, torch.logsumexp(x, -1), torch.zeros((), dtype=torch.float64, device=d)) \
                        if kv else torch.zeros(x.shape[:2], dtype=torch.float64, device=d)
                    p = torch.exp(x - z[..., None]) * some[..., None]
                    o, A = p @ V, p @ V.abs()
                    e = (2 * E + 2 * SMALL + u + 2 * kv * 2.0 ** -23)[..., None] * A + u * o.abs()
                    if self.dtype == torch.float16:
                        vis = torch.einsum("tj,jd->td", seen.double(), V.abs())[:, None, :]
                        e = e + 2.0 ** -25 * vis + 2.0 ** -25
                    out[rows, hs], tol[rows, hs] = o, e + 1e-38
                    lse[rows, hs] = torch.where(some, z, torch.full_like(z, -math.inf))
                    ltol[rows, hs] = E + SMALL + (kv + 8) * 2.0 ** -23 + z.abs() * 2.0 ** -22
        return out, tol, lse, ltol

    def check(self, out, lse):
        torch = T()
        R = self.starts[-1]
        ref, tol, rl, ltol = self.reference()
        got = out[:R].double()
        assert torch.isfinite(got).all()
        bad = (got - ref).abs() > tol
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), float(((got - ref).abs() / tol).max()))
        none = torch.isinf(rl)
        assert torch.equal(torch.isneginf(lse[:R]), none)
        dl = (lse[:R].double() - rl)[~none].abs()
        assert (dl <= ltol[~none]).all(), float((dl / ltol[~none]).max())


def dt(name):
    return getattr(T(), {"f16": "float16", "bf16": "bfloat16"}[name])


HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (4, 4, 64), (16, 1, 128), (65, 1, 64), (128, 1, 64), (3, 3, 128)]
# (new tokens, cached keys): single tokens, tile and page edges, empty sequences,
# rows that see no key (more new tokens than keys), sequences without new tokens
RAGGED = [
    [(1, 1)],
    [(1, 64), (1, 65), (1, 63), (1, 128), (1, 129), (1, 0), (1, 700)],
    [(0, 0), (5, 5), (0, 70), (3, 200), (18, 18), (19, 19), (9, 127), (36, 300), (37, 37)],
    [(7, 3), (1, 0), (40, 1), (2, 2)],
    [(130, 130), (1, 513), (64, 64), (257, 385), (0, 9)],
    [(2, 2), (4, 130), (0, 5), (3, 64), (1, 65), (4, 1), (2, 1200)],
    [(2, 40), (1, 1100), (2, 127)],
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("seqs", RAGGED, ids=range(len(RAGGED)))
def test_attention_ragged(vv, seqs, heads, dtype):
    c = Chunk(seqs, heads, dt(dtype), seed=sum(heads)).gpu()
    c.check(*c.attend())


@pytest.mark.parametrize("seqs,heads", [([(1, 9001)], (28, 4, 128)), ([(3, 5000), (1, 4097)], (14, 2, 64)),
                                        ([(700, 4000)], (12, 2, 128)), ([(33, 2500), (300, 300)], (28, 4, 128)),
                                        ([(1, 64 + 31 * s) for s in range(70)], (14, 2, 64)),
                                        ([(2000, 2000)], (14, 2, 64))])
def test_attention_long(vv, seqs, heads):
    """Few long rows (spread over the GPU through the workspace), also with a
    workspace that is missing or too small for that, and many short rows."""
    torch = T()
    c = Chunk(seqs, heads, torch.float16, seed=5).gpu()
    c.check(*c.attend())
    lib, p = vv.lib(), c.pages._p
    need = lib.vvq2_attention_paged_workspace(p, c.total, c.max_q, c.max_kv, c.nq)
    for n in (0, need // 3 // 16 * 16, need):
        ws = torch.empty(max(16, n), dtype=torch.uint8, device="cuda:0")
        out, lse = torch.empty_like(c.qd), torch.empty(c.qd.shape[:2], device="cuda:0")
        w = c.nq * c.hd
        rc = lib.vvq2_attention_paged(p, 0, c.qd.data_ptr(), w, c.qs.data_ptr(), c.kl.data_ptr(), c.total, c.max_q,
                                      c.max_kv, c.nq, c.scale, out.data_ptr(), w, lse.data_ptr(),
                                      ws.data_ptr() if n else None, n, None,
                                      torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        c.check(out, lse)


@pytest.mark.parametrize("seqs", [[(1, 27), (2, 300), (1, 1500)], [(1, 5000)], [(40, 700), (7, 3000)],
                                  [(n, n + 90) for n in (1, 5, 17, 18, 37, 200, 601)] * 8])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=["64", "128"])
def test_attention_in_place(vv, seqs, heads):
    """out may be q itself."""
    torch = T()
    c = Chunk(seqs, heads, torch.float16, seed=16).gpu()
    want, want_lse = c.attend()
    out, lse = c.attend(out=c.qd)
    assert out is c.qd
    c.check(out, lse)
    assert torch.equal(out, want)
    assert torch.equal(lse, want_lse)


@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128)], ids=["64", "128"])
def test_attention_repeats_to_the_bit(vv, heads):
    """More items than blocks, so which block has which is left to the hardware."""
    torch = T()
    c = Chunk([(n, n + 90) for n in (5, 17, 18, 37, 200, 601)] * 10, heads, torch.float16, seed=17).gpu()
    want, want_lse = c.attend()
    for _ in range(8):
        out, lse = c.attend()
        assert torch.equal(out, want)
        assert torch.equal(lse, want_lse)
    weights = [vvq2.attention_key_weights(c.qd, want_lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv) for _ in range(8)]
    assert all(torch.equal(w, weights[0]) for w in weights)


@pytest.mark.parametrize("seqs", [RAGGED[2], [(1, 3000), (2, 40)]])
def test_attention_bounds_may_be_loose(vv, seqs):
    """max_q and max_kv are upper bounds; table entries past a sequence's pages are never read."""
    torch = T()
    c = Chunk(seqs, (14, 2, 64), torch.float16, seed=6).gpu()
    c.max_q, c.max_kv = 4000, c.bt.shape[1] * PAGE
    err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    c.check(*c.attend(err=err))
    assert err.item() == 0


def test_attention_padding_strides_and_given_buffers(vv):
    """Rows behind the last sequence and the gaps of strided outputs keep what
    they held; q may be a slice of a fused projection."""
    torch = T()
    c = Chunk([(3, 50), (20, 20), (1, 300)], (12, 2, 128), torch.float16, seed=3, pad=5).gpu()
    w = c.nq * c.hd
    fused = torch.full((c.total, w + 2 * 2 * 128), 7.0, dtype=torch.float16, device="cuda:0")
    fused[:, :w] = c.qd.reshape(c.total, w)
    q = fused[:, :w].unflatten(1, (c.nq, c.hd))
    hold = torch.full((c.total, w + 64), 5.0, dtype=torch.float16, device="cuda:0")
    out = hold[:, 64:].unflatten(1, (c.nq, c.hd))
    lse = torch.full((c.total, c.nq), 9.0, device="cuda:0")
    r = vv.attention_paged(q, c.pages, c.qs, c.kl, c.max_q, c.max_kv, out=out, lse=lse)
    assert r[0] is out and r[1] is lse
    c.check(out, lse)
    assert (hold[:, :64] == 5).all() and (out[-5:] == 5).all() and (lse[-5:] == 9).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_nonfinite_values_behind_the_mask(vv, bad, dtype):
    """A non-finite V element of a later token reaches the rows that see it and
    no others; a non-finite K row likewise."""
    torch = T()
    seqs, j, d = [(100, 230), (1, 65)], 190, 17
    c = Chunk(seqs, (14, 2, 64), dt(dtype), seed=8)
    clean = Chunk(seqs, (14, 2, 64), dt(dtype), seed=8).gpu()
    ref, lref = clean.attend()
    c.V[c.bt[0, j // PAGE], 1, j % PAGE, d] = bad
    got, lse = c.gpu().attend()
    first = j - 130                                   # the first token that sees key j
    assert torch.equal(got[:first], ref[:first]) and torch.equal(got[100:], ref[100:])
    assert torch.equal(got[:, :7], ref[:, :7]) and torch.equal(lse, lref)
    hit = got[first:100, 7:]
    assert (torch.isnan(hit[..., d]) if bad != bad else hit[..., d] == bad).all()
    hit, cln = hit.clone(), ref[first:100, 7:].clone()
    hit[..., d] = cln[..., d] = 0
    assert torch.equal(hit, cln)

    c = Chunk(seqs, (14, 2, 64), dt(dtype), seed=8)
    c.K[c.bt[0, j // PAGE], 0, j % PAGE] = float("nan")
    got, lse = c.gpu().attend()
    assert torch.equal(got[:first], ref[:first]) and torch.equal(got[100:], ref[100:])
    assert torch.equal(got[:, 7:], ref[:, 7:])
    assert torch.isnan(got[first:100, :7]).all() and torch.isnan(lse[first:100, :7]).all()


@pytest.mark.parametrize("kv", [70, 3000])
@pytest.mark.parametrize("heads,n", [((14, 2, 64), 2), ((12, 2, 128), 5)])
def test_attention_nonfinite_values_few_rows(vv, heads, n, kv):
    """The same for a few drafted tokens, one page or many: +inf, -inf and NaN
    in different columns, +inf and -inf in one."""
    torch = T()
    make = lambda: Chunk([(n, kv), (1, 9)], heads, torch.float16, seed=14)
    ref, lref = make().gpu().attend()
    c = make()
    G, j = heads[0] // heads[1], kv - 1               # the last token's own key
    at = (c.bt[0, j // PAGE], 0, j % PAGE)
    c.V[(*at, 3)], c.V[(*at, 4)], c.V[(*at, 5)] = float("inf"), float("-inf"), float("nan")
    c.V[(*at, 6)] = float("inf")
    if n > 2:
        c.V[c.bt[0, (j - 1) // PAGE], 0, (j - 1) % PAGE, 6] = float("-inf")   # token n - 2's
    got, lse = c.gpu().attend()
    assert torch.equal(lse, lref) and torch.equal(got[:n - 2], ref[:n - 2]) and torch.equal(got[n:], ref[n:])
    assert torch.equal(got[:, G:], ref[:, G:])
    hit = got[n - 1, :G]
    assert (hit[:, 3] == float("inf")).all() and (hit[:, 4] == float("-inf")).all() and torch.isnan(hit[:, 5]).all()
    if n > 2:
        assert torch.isnan(hit[:, 6]).all() and (got[n - 2, :G, 6] == float("-inf")).all()
    else:
        assert (hit[:, 6] == float("inf")).all()
    assert torch.equal(hit[:, 7:], ref[n - 1, :G, 7:]) and torch.equal(hit[:, :3], ref[n - 1, :G, :3])


def test_attention_all_scores_minus_infinity(vv):
    """A row whose only visible score is -inf sums to nothing: out 0, lse -inf."""
    torch = T()
    c = Chunk([(2, 2)], (4, 4, 64), torch.float16, seed=2)
    c.q.fill_(1.0)
    c.K[c.bt[0, 0], :, 0] = 0
    c.K[c.bt[0, 0], :, 0, 0] = float("-inf")
    out, lse = c.gpu().attend()
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all()
    assert torch.allclose(out[1].cpu().float(), c.vals[0][1].float())   # the second key alone: exact


def test_attention_large_scores(vv):
    """Scores of several hundred: the running maximum keeps every exponent in range."""
    torch = T()
    c = Chunk([(40, 600), (1, 1000)], (14, 2, 64), torch.float16, seed=4, qscale=60.0).gpu()
    out, lse = c.attend()
    c2 = Chunk([(40, 600), (1, 1000)], (14, 2, 64), torch.float16, seed=4, qscale=60.0)
    ref, tol, rl, ltol = c2.reference()
    # scores to ~2^10: their f32 roundings are 8 times the header's 2^-17
    assert ((out.double() - ref).abs() <= 8 * tol).all() and ((lse.double() - rl).abs() <= 8 * ltol).all()


def test_attention_error_words(vv):
    torch = T()
    c = Chunk([(2, 200), (1, 90)], (14, 2, 64), torch.float16, seed=9).gpu()
    good = c.attend()
    err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    c.attend(err=err)
    assert err.item() == 0
    # a length beyond max_kv is cut to it
    c.kl[0] = 1200
    got = c.attend(err=err)
    assert err.item() == 5 and torch.equal(got[0], good[0])
    # an entry that names no page stands for a page of zeros
    c.kl[0] = 200
    for entry in (-1, c.pages.n_pages, 1 << 30):
        err.zero_()
        old = c.pages.block_table[1, 0].item()
        c.pages.block_table[1, 0] = entry
        got = c.attend(err=err)
        c.pages.block_table[1, 0] = old
        assert err.item() == 6 and torch.equal(got[0][:2], good[0][:2])
        z = Chunk([(2, 200), (1, 90)], (14, 2, 64), torch.float16, seed=9)
        z.K[z.bt[1, 0]] = 0
        z.V[z.bt[1, 0]] = 0
        ref = z.gpu().attend()
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    # q_start that runs past the rows is cut
    err.zero_()
    c.qs[2] = 50
    got = c.attend(err=err)
    assert err.item() == 5 and torch.equal(got[0], good[0])


def test_attention_key_offsets_past_32_bits(vv):
    """Pages beyond 2^31 elements of a pool."""
    torch = T()
    n_pages, nkv, hd = 33500, 8, 128
    k = torch.empty((n_pages, nkv, PAGE, hd), dtype=torch.float16, device="cuda:0")
    v = torch.empty_like(k)
    c = Chunk([(5, 150), (1, 64)], (16, 8, 128), torch.float16, seed=11)
    at = torch.randperm(700, generator=torch.Generator().manual_seed(1))[:c.K.shape[0]] + n_pages - 700
    at[0] = n_pages - 1
    k[at] = c.K.cuda()
    v[at] = c.V.cuda()
    c.bt = torch.where(c.bt >= 0, at[c.bt.clamp(min=0).long()].int(), c.bt)
    c.gpu()
    c.pages = vv.Pages(k, v, c.bt.cuda())
    out, lse = c.attend()
    c.check(out, lse)
    w = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    check_weights(c, lse, w, None)


def test_attention_streams_graphs_and_repeats(vv):
    """Same bits from repeated calls, on another stream, and from a replayed
    graph whose lengths, table and inputs changed; two graphs side by side."""
    torch = T()
    a = Chunk([(1, 3000), (4, 700)], (14, 2, 64), torch.float16, seed=12).gpu()
    b = Chunk([(1, 2500), (4, 500)], (14, 2, 64), torch.float16, seed=13)
    ref = a.attend()
    for _ in range(3):
        again = a.attend()
        assert torch.equal(ref[0], again[0]) and torch.equal(ref[1], again[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = a.attend(stream=s)
    s.synchronize()
    assert torch.equal(ref[0], other[0])
    other = a.attend(stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(ref[0], other[0])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = a.attend()
            w = vv.attention_key_weights(a.qd, r[1], a.pages, a.qs, a.kl, a.max_q, a.max_kv)
        graphs.append((g, r, w))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for (g, _, _), st in zip(graphs, (s1, s2)):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for _, r, _ in graphs:
        assert torch.equal(ref[0], r[0]) and torch.equal(ref[1], r[1])
    # other contents in the same buffers
    a.pages.k[:b.K.shape[0]] = b.K.cuda()
    a.pages.v[:b.V.shape[0]] = b.V.cuda()
    a.pages.block_table.fill_(-1)
    a.pages.block_table[:, :b.bt.shape[1]] = b.bt.cuda()
    a.qd.copy_(b.q)
    a.kl.copy_(torch.tensor([2500, 500], dtype=torch.int32))
    b.gpu()
    g, r, w = graphs[1]
    g.replay()
    torch.cuda.synchronize()
    b.check(*r)
    check_weights(b, r[1], w, None)


def check_weights(c, lse, got, w_in, prior=None):
    """got against the definition; prior: what w_out held (words past the keys)."""
    torch = T()
    d = "cuda:0"
    for s, (n, kv) in enumerate(c.seqs):
        for g in range(c.nkv):
            hs, rows = slice(g * c.G, (g + 1) * c.G), slice(c.starts[s], c.starts[s] + n)
            q, K = c.q[rows, hs].to(d).double(), c.keys[s][:, g].to(d).double()
            x = torch.einsum("thd,jd->thj", q, K) * c.scale
            E = c.hd * 2.0 ** -23 * c.scale * torch.einsum("thd,jd->thj", q.abs(), K.abs())
            seen = torch.arange(kv, device=d)[None, :] < (kv - n + torch.arange(n, device=d) + 1)[:, None]
            seen = seen[:, None, :].expand_as(x)
            l = lse[rows, hs].double()[..., None]
            p = torch.where(seen, torch.exp(x - l), torch.zeros_like(x))
            w = p.sum((0, 1))
            # the exponent's error E plus a few f32 roundings of x and lse, and
            # the f32 sum over the rows
            tol = ((E + SMALL + l.abs().nan_to_num(0, 0, 0) * 2.0 ** -22) * p).sum((0, 1)) + \
                w * (n * c.G + 8) * 2.0 ** -23 + 1e-30
            if w_in is not None:
                old = torch.arange(kv, device=d) < kv - n
                w = torch.where(old, w + w_in[s, g, :kv].double(), w)
                tol = tol + w.abs() * 2.0 ** -23
            e = (got[s, g, :kv].double() - w).abs()
            assert (e <= tol).all(), (s, g, float((e / tol).max()), int((e / tol).argmax()))
            if prior is not None:
                assert torch.equal(got[s, g, kv:], prior[s, g, kv:])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("seqs", RAGGED, ids=range(len(RAGGED)))
def test_key_weights(vv, seqs, heads, dtype):
    torch = T()
    c = Chunk(seqs, heads, dt(dtype), seed=20 + sum(heads)).gpu()
    _, lse = c.attend()
    if not c.max_kv:
        return
    width = c.max_kv + 5
    prior = torch.randn((len(seqs), c.nkv, width), device="cuda:0")
    w_in = torch.rand((len(seqs), c.nkv, width), device="cuda:0")
    got = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv, w_out=prior.clone())
    check_weights(c, lse, got, None, prior)
    got = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv, w_in=w_in, w_out=prior.clone())
    check_weights(c, lse, got, w_in, prior)
    both = w_in.clone()
    same = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv, w_in=both, w_out=both)
    assert same is both
    for s, (_, kv) in enumerate(seqs):
        assert torch.equal(both[s, :, :kv], got[s, :, :kv]) and torch.equal(both[s, :, kv:], w_in[s, :, kv:])


@pytest.mark.parametrize("seqs,heads", [([(32, 5000)], (28, 4, 128)),
                                        ([(1, 64 + 29 * s) for s in range(40)], (14, 2, 64)),
                                        ([(900, 1500), (1, 1)], (12, 2, 128))])
def test_key_weights_long(vv, seqs, heads):
    """Also: the weights of all keys add up to one per (row, head)."""
    torch = T()
    c = Chunk(seqs, heads, torch.float16, seed=31, pad=3).gpu()
    _, lse = c.attend()
    got = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    check_weights(c, lse, got, None)
    for s, (n, kv) in enumerate(seqs):
        want = n * c.G
        # each row's probabilities add up to one within its lse's error (the
        # bound of check), here E <= hd * 2^-23 * scale * sum |q k| < 2^-12
        assert ((got[s, :, :kv].double().sum(-1) - want).abs() <= want * 2.0 ** -11).all()


def test_key_weights_long_rows_in_chunks(vv):
    """Rows enough for many chunks: taken in any order by the blocks, added up
    in one; with workspaces too small for that; captured and replayed."""
    torch = T()
    c = Chunk([(300, 300), (5, 900), (0, 40)], (128, 1, 64), torch.float16, seed=35).gpu()
    _, lse = c.attend()
    got = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    check_weights(c, lse, got, None)
    w_in = torch.rand_like(got)
    added = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv, w_in=w_in,
                                     w_out=torch.zeros_like(got))
    check_weights(c, lse, added, w_in)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    for _ in range(3):
        again.fill_(-1.0)
        g.replay()
        torch.cuda.synchronize()
        for s, (_, kv) in enumerate(c.seqs):
            assert torch.equal(again[s, :, :kv], got[s, :, :kv])
    lib, p = vv.lib(), c.pages._p
    need = lib.vvq2_attention_key_weights_workspace(p, c.total, c.max_q, c.max_kv, c.nq)
    assert need > 0
    for n in (0, 8, need // 4 // 16 * 16, need // 2 // 16 * 16, need):
        ws = torch.empty(max(16, n), dtype=torch.uint8, device="cuda:0")
        out = torch.zeros_like(got)
        rc = lib.vvq2_attention_key_weights(p, 0, c.qd.data_ptr(), c.nq * c.hd, lse.data_ptr(), c.qs.data_ptr(),
                                            c.kl.data_ptr(), c.total, c.max_q, c.max_kv, c.nq, c.scale, None,
                                            out.data_ptr(), out.shape[2], ws.data_ptr() if n else None, n, None,
                                            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        check_weights(c, lse, out, None)


def test_no_rows_at_all(vv):
    """No new token in any sequence: older keys keep their weights, without any
    they are 0; a call without a key does nothing."""
    torch = T()
    c = Chunk([(0, 70), (0, 0), (0, 300)], (14, 2, 64), torch.float16, seed=36).gpu()
    out, lse = c.attend()
    assert out.shape == (0, 14, 64) and lse.shape == (0, 14)
    w_in = torch.rand((3, 2, 300), device="cuda:0")
    got = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, 0, 300, w_in=w_in, w_out=torch.full_like(w_in, 5.0))
    zero = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, 0, 300, w_out=torch.full_like(w_in, 5.0))
    for s, n in enumerate((70, 0, 300)):
        assert torch.equal(got[s, :, :n], w_in[s, :, :n]) and (got[s, :, n:] == 5).all()
        assert (zero[s, :, :n] == 0).all() and (zero[s, :, n:] == 5).all()
    c.kl.zero_()
    assert (vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, 0, 0, w_out=w_in.clone()) == w_in).all()


def test_key_weights_error_words_and_masked_keys(vv):
    torch = T()
    c = Chunk([(3, 130), (5, 5)], (14, 2, 64), torch.float16, seed=33)
    c.K[c.bt[0, 2], :, 1] = float("nan")          # the last token's own key: only its rows see it
    c.gpu()
    clean = Chunk([(3, 130), (5, 5)], (14, 2, 64), torch.float16, seed=33).gpu()
    _, lse = clean.attend()
    err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    a = vv.attention_key_weights(clean.qd, lse, clean.pages, c.qs, c.kl, 5, 130, err=err)
    b = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, 5, 130, err=err)
    assert err.item() == 0
    assert torch.equal(a[0, :, :129], b[0, :, :129]) and torch.equal(a[1], b[1]) and torch.isnan(b[0, :, 129]).all()
    # NaN queries of another sequence stay out
    q = c.qd.clone()
    q[3:] = float("nan")
    b = vv.attention_key_weights(q, lse, clean.pages, c.qs, c.kl, 5, 130)
    assert torch.equal(a[0], b[0])
    clean.kl[0] = 9999
    vv.attention_key_weights(clean.qd, lse, clean.pages, clean.qs, clean.kl, 5, 130, err=err)
    assert err.item() == 5
    clean.kl[0] = 130
    err.zero_()
    clean.pages.block_table[0, 1] = -7
    vv.attention_key_weights(clean.qd, lse, clean.pages, clean.qs, clean.kl, 5, 130, err=err)
    assert err.item() == 6


# ------------------------------------------------------------------ eviction
def evict_ref(w, n, keep, first, recent):
    if n <= keep:
        return list(range(n))
    x = w[:n].double().tolist()
    mid = sorted(range(first, n - recent), key=lambda j: (x[j] != x[j], -x[j] if x[j] == x[j] else 0, j))
    return sorted(list(range(first)) + list(range(n - recent, n)) + mid[:keep - first - recent])


def run_evict(vv, lens, keep, first, recent, nkv=2, hd=64, layers=1, dtype="f16", weights=None, seed=1, max_kv=None,
              width=None):
    torch = T()
    rng = torch.Generator().manual_seed(seed)
    src, n_src = table(lens, rng)
    dst, n_dst = table([min(l, keep) for l in lens], rng, first=n_src)
    shape = (layers, n_src + n_dst, nkv, PAGE, hd)
    k = torch.randint(0, 0x7000, shape, generator=rng, dtype=torch.int16).view(dt(dtype)).cuda()
    v = torch.randint(0, 0x7000, shape, generator=rng, dtype=torch.int16).view(dt(dtype)).cuda()
    width = max(1, max(lens)) if width is None else width
    w = torch.rand((layers, len(lens), nkv, width), generator=rng)
    if weights is not None:
        w = weights(w)
    k0, v0 = k.clone(), v.clone()
    lead = (layers, len(lens), nkv, keep)
    kept = torch.full(lead, -9, dtype=torch.int32, device="cuda:0")
    w_out = torch.full(lead, 123.0, device="cuda:0")
    err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    kl = torch.tensor(lens, dtype=torch.int32, device="cuda:0")
    got = vv.pages_evict(vv.Pages(k, v, src.cuda()), dst.cuda(), kl, w.cuda(), keep, first, recent, max_kv=max_kv,
                         kept=kept, w_out=w_out, err=err)
    assert got[0] is kept and got[2] is w_out and err.item() == 0
    assert got[1].tolist() == [min(l, keep) for l in lens]
    want_k, want_v = k0, v0
    kc, wc = kept.cpu(), w_out.cpu()
    for l in range(layers):
        for s, n in enumerate(lens):
            for g in range(nkv):
                ref = evict_ref(w[l, s, g], n, keep, first, recent)
                m = len(ref)
                assert kc[l, s, g].tolist() == ref + [-1] * (keep - m), (l, s, g)
                j, i = torch.tensor(ref, dtype=torch.long), torch.arange(m)
                assert torch.equal(wc[l, s, g, :m].view(torch.int32), w[l, s, g, j].view(torch.int32))
                assert (wc[l, s, g, m:] == 123).all()
                sp, dp = src[s, j // PAGE].long().cuda(), dst[s, i // PAGE].long().cuda()
                j, i = j.cuda(), i.cuda()
                want_k[l, dp, g, i % PAGE] = k0[l, sp, g, j % PAGE]
                want_v[l, dp, g, i % PAGE] = v0[l, sp, g, j % PAGE]
    # the kept rows bit for bit, and every other row of the pools untouched
    assert torch.equal(k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), want_v.view(torch.int16))


@pytest.mark.parametrize("lens,keep,first,recent", [
    ([1], 1, 0, 0), ([0, 1, 2], 1, 0, 1), ([5, 0, 200], 64, 3, 60), ([64, 65, 63, 128, 129], 64, 0, 0),
    ([300, 100], 100, 100, 0), ([300, 100], 100, 0, 100), ([1000, 999, 31], 257, 13, 50), ([130], 129, 1, 127),
    ([2500, 2049, 2048, 2047, 1025, 1023], 1024, 4, 100), ([4097], 1000, 0, 0), ([700], 5000, 100, 100)])
@pytest.mark.parametrize("shape", [dict(nkv=2, hd=64), dict(nkv=1, hd=128, layers=3, dtype="bf16")],
                         ids=["64", "128x3"])
def test_evict(vv, lens, keep, first, recent, shape):
    run_evict(vv, lens, keep, first, recent, **shape)


def quantized(w):
    return (w * 6).floor() / 6                     # many equal weights


def zeros(w):
    return w * 0


def mixed(w):
    w = (w - 0.5) * 4
    w.flatten()[::7] = float("nan")
    w.flatten()[1::5] = 0.0
    w.flatten()[2::5] = -0.0                       # equal to +0
    w.flatten()[3::11] = float("inf")
    w.flatten()[4::13] = float("-inf")
    return w


def all_nan(w):
    return w * float("nan")


def tiny(w):
    return (w * 2.0 ** 20).floor() * 2.0 ** -149 * 8   # subnormals


@pytest.mark.parametrize("weights", [quantized, zeros, mixed, all_nan, tiny])
@pytest.mark.parametrize("lens,keep,first,recent", [([500, 257, 31], 128, 5, 20), ([3001], 1500, 0, 1),
                                                    ([40000], 30000, 128, 1024), ([60001, 700], 600, 50, 550),
                                                    ([51201], 51000, 0, 0)])
def test_evict_ties_and_special_weights(vv, lens, keep, first, recent, weights):
    run_evict(vv, lens, keep, first, recent, weights=weights, seed=3)


def test_evict_weights_wider_than_the_keys(vv):
    run_evict(vv, [200, 150], 100, 7, 8, width=333, max_kv=200)
    run_evict(vv, [200, 150], 100, 7, 8, width=333)


def test_evict_error_words_and_bad_pages(vv):
    torch = T()
    rng = torch.Generator().manual_seed(2)
    src, n_src = table([300, 100], rng)
    dst, n_dst = table([130, 100], rng, first=n_src)
    k = torch.randn((n_src + n_dst, 2, PAGE, 64), generator=rng).half().cuda()
    v = torch.randn((n_src + n_dst, 2, PAGE, 64), generator=rng).half().cuda()
    w = torch.rand((2, 2, 300), generator=rng).cuda()
    kl = torch.tensor([300, 100], dtype=torch.int32, device="cuda:0")
    err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    k1, v1 = k.clone(), v.clone()
    good = vv.pages_evict(vv.Pages(k1, v1, src.cuda()), dst.cuda(), kl, w, 130, 10, 20, err=err)
    assert err.item() == 0
    # a destination that names no page: its rows are dropped, the rest moves
    bad = dst.clone()
    bad[0, 1] = n_src + n_dst
    k2, v2 = k.clone(), v.clone()
    got = vv.pages_evict(vv.Pages(k2, v2, src.cuda()), bad.cuda(), kl, w, 130, 10, 20, err=err)
    assert err.item() == 6 and torch.equal(got[0], good[0])
    lost = dst[0, 1].item()
    k1[lost], v1[lost] = k[lost], v[lost]
    assert torch.equal(k1, k2) and torch.equal(v1, v2)
    # a source that names none: zeros
    err.zero_()
    bad = src.clone()
    bad[1, 0] = -3
    k2, v2 = k.clone(), v.clone()
    vv.pages_evict(vv.Pages(k2, v2, bad.cuda()), dst.cuda(), kl, w, 130, 10, 20, err=err)
    assert err.item() == 6 and (k2[dst[1, 0]] == 0).all() and (v2[dst[1, 0]] == 0).all()
    # a length beyond max_kv is cut
    err.zero_()
    kl[0] = 5000
    k2, v2 = k.clone(), v.clone()
    got = vv.pages_evict(vv.Pages(k2, v2, src.cuda()), dst.cuda(), kl, w, 130, 10, 20, err=err)
    assert err.item() == 5 and torch.equal(got[0], good[0]) and torch.equal(got[1], good[1])


def test_evict_shared_source_pages_and_graph(vv):
    """Two sequences that share their pages; captured, replayed after the weights changed."""
    torch = T()
    rng = torch.Generator().manual_seed(4)
    src, n_src = table([400], rng)
    src = src.repeat(2, 1)
    dst, n_dst = table([128, 128], rng, first=n_src)
    k = torch.randn((n_src + n_dst, 2, PAGE, 64), generator=rng).half().cuda()
    v = torch.randn((n_src + n_dst, 2, PAGE, 64), generator=rng).half().cuda()
    pages, dst_d = vv.Pages(k, v, src.cuda()), dst.cuda()
    kl = torch.tensor([400, 400], dtype=torch.int32, device="cuda:0")
    w = torch.rand((2, 2, 400), device="cuda:0")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept, new_len, w_out = vv.pages_evict(pages, dst_d, kl, w, 128, 4, 30)
    for seed in (1, 2):
        w.copy_(torch.rand((2, 2, 400), generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        assert new_len.tolist() == [128, 128]
        for s in range(2):
            for h in range(2):
                ref = evict_ref(w[s, h].cpu(), 400, 128, 4, 30)
                assert kept[s, h].tolist() == ref
                j = torch.tensor(ref)
                i = torch.arange(128)
                assert torch.equal(k[dst[s, i // PAGE].long().cuda(), h, (i % PAGE).cuda()],
                                   k[src[s, j // PAGE].long().cuda(), h, (j % PAGE).cuda()])


def test_evict_without_weights_out(vv):
    torch = T()
    rng = torch.Generator().manual_seed(6)
    src, n_src = table([90], rng)
    dst, n_dst = table([40], rng, first=n_src)
    k = torch.randn((n_src + n_dst, 1, PAGE, 64), generator=rng).half().cuda()
    v = torch.randn((n_src + n_dst, 1, PAGE, 64), generator=rng).half().cuda()
    w = torch.rand((1, 1, 90), generator=rng).cuda()
    pages, kl, dst = vv.Pages(k, v, src.cuda()), torch.tensor([90], dtype=torch.int32, device="cuda:0"), dst.cuda()
    ref = vv.pages_evict(pages, dst, kl, w, 40, 3, 7)
    kept, new_len = torch.zeros_like(ref[0]), torch.zeros_like(ref[1])
    rc = vv.lib().vvq2_pages_evict(pages._p, dst.data_ptr(), dst.shape[1], kl.data_ptr(), 90, w.data_ptr(), 90, 40, 3,
                                   7, kept.data_ptr(), None, new_len.data_ptr(), None,
                                   torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(kept, ref[0]) and torch.equal(new_len, ref[1])


# ----------------------------------------------------------- refusals, on a GPU
def test_refusals_of_memory_that_is_not_on_the_gpu(vv):
    torch = T()
    c = Chunk([(2, 20)], (14, 2, 64), torch.float16).gpu()
    host = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(vv.VVQ2Error) as e:
        vv.attention_paged(c.qd, c.pages, host, c.kl, 2, 20)
    assert e.value.rc == -2
    with pytest.raises(vv.VVQ2Error):
        vv.attention_paged(c.qd.cpu(), c.pages, c.qs, c.kl, 2, 20)
    with pytest.raises(vv.VVQ2Error):
        vv.attention_paged(c.qd, c.pages, c.qs, c.kl, 2, 20, scale=0.0)
    with pytest.raises(vv.VVQ2Error):
        vv.attention_paged(c.qd, c.pages, c.qs, c.kl, 2, 20, layer=1)
    with pytest.raises(vv.VVQ2Error):
        vv.attention_paged(c.qd, c.pages, c.qs, c.kl, 2, 20, err=torch.zeros(1, dtype=torch.int32))
    pinned = torch.zeros(1, dtype=torch.int32).pin_memory()
    c.attend(err=pinned)
    torch.cuda.synchronize()
    assert pinned.item() == 0
    # the context is as good as before
    c.check(*c.attend())


# --------------------------------------------------------------------- together
@pytest.mark.parametrize("heads,dtype", [((14, 2, 64), "f16"), ((28, 4, 128), "bf16")])
def test_streams_attend_weigh_evict_and_go_on(vv, heads, dtype):
    """Two layers of three streams: prompts in one packed call, weights gathered
    over the prompt and some decoded tokens, an eviction to a budget, and
    decoding on the shortened pages; every step against the same steps in 64
    bits on per-head key lists."""
    torch = T()
    nq, nkv, hd = heads
    G, layers, keep, first, recent = nq // nkv, 2, 150, 8, 40
    rng = torch.Generator().manual_seed(77)
    prompts = [260, 97, 171]
    cap = [(n + 12 + PAGE) // PAGE for n in prompts]
    per = max(cap) + 1
    n_pages = 3 * per + 3 * 4
    D = dt(dtype)
    k = torch.full((layers, n_pages, nkv, PAGE, hd), float("nan"), dtype=D, device="cuda:0")
    v = torch.full_like(k, float("nan"))
    perm = torch.randperm(n_pages, generator=rng).int()
    bt, dst = perm[:3 * per].reshape(3, per).cuda(), perm[3 * per:].reshape(3, 4).cuda()
    width = per * PAGE
    w = torch.zeros((layers, 3, nkv, width), device="cuda:0")
    hist = [[[([], []) for _ in range(nkv)] for _ in range(3)] for _ in range(layers)]   # key / value lists
    wref = [[[[] for _ in range(nkv)] for _ in range(3)] for _ in range(layers)]
    scale = hd ** -0.5
    u = torch.finfo(D).eps / 2

    def step(tab, lens, new, w, check_w=True):
        pages = vv.Pages(k, v, tab)
        total = sum(new)
        qs = torch.tensor([sum(new[:i]) for i in range(4)], dtype=torch.int32, device="cuda:0")
        kl = torch.tensor([a + b for a, b in zip(lens, new)], dtype=torch.int32, device="cuda:0")
        max_q, max_kv = max(new), max(a + b for a, b in zip(lens, new))
        for l in range(layers):
            q = (torch.randn((total, nq, hd), generator=rng) * 2).to(D)
            kn = torch.randn((total, nkv, hd), generator=rng).to(D)
            vn = torch.randn((total, nkv, hd), generator=rng).to(D)
            at = 0
            for s in range(3):
                for t in range(new[s]):
                    p = lens[s] + t
                    k[l, tab[s, p // PAGE], :, p % PAGE] = kn[at].cuda()
                    v[l, tab[s, p // PAGE], :, p % PAGE] = vn[at].cuda()
                    for g in range(nkv):
                        hist[l][s][g][0].append(kn[at, g].double())
                        hist[l][s][g][1].append(vn[at, g].double())
                        wref[l][s][g].append(0.0)
                    at += 1
            qd = q.cuda()
            out, lse = vv.attention_paged(qd, pages, qs, kl, max_q, max_kv, layer=l, want_lse=True)
            vv.attention_key_weights(qd, lse, pages, qs, kl, max_q, max_kv, w_in=w[l], w_out=w[l], layer=l)
            out = out.double().cpu()
            at = 0
            for s in range(3):
                n, L = new[s], lens[s] + new[s]
                for g in range(nkv):
                    K, V = torch.stack(hist[l][s][g][0]), torch.stack(hist[l][s][g][1])
                    x = torch.einsum("thd,jd->thj", q[at:at + n, g * G:(g + 1) * G].double(), K) * scale
                    see = torch.arange(L)[None, :] < (lens[s] + torch.arange(n) + 1)[:, None]
                    x = x.masked_fill(~see[:, None], -math.inf)
                    p = torch.softmax(x, -1)
                    ref, A = p @ V, p @ V.abs()
                    # 2^-12 covers 2E + 2 * 2^-17 + n * 2^-22 here: E <= hd * 2^-23 * scale *
                    # sum |q k| <= 128 * 2^-23 * 2^-3.5 * 2^8 < 2^-11.5 at its worst element,
                    # 2^-13 at these inputs' (sum |q k| < 2^8 * 0.7 for N(0, 2) x N(0, 1))
                    tol = (u + 2.0 ** -12) * A + u * ref.abs() + 2.0 ** -20
                    assert ((out[at:at + n, g * G:(g + 1) * G] - ref).abs() <= tol).all()
                    wr = torch.tensor(wref[l][s][g], dtype=torch.float64) + p.sum((0, 1))
                    wref[l][s][g] = wr.tolist()
                    e = (w[l, s, g, :L].double().cpu() - wr).abs()
                    assert (e <= wr * 2.0 ** -11 + 1e-12).all()
                at += n
        return [a + b for a, b in zip(lens, new)]

    lens = step(bt, [0, 0, 0], prompts, w)
    for _ in range(2):
        lens = step(bt, lens, [1, 2, 1], w)
    kl = torch.tensor(lens, dtype=torch.int32, device="cuda:0")
    kept, new_len, w_kept = vv.pages_evict(vv.Pages(k, v, bt), dst, kl, w, keep, first, recent, max_kv=max(lens))
    assert new_len.tolist() == [min(n, keep) for n in lens]
    kept_c = kept.cpu()
    for l in range(layers):
        for s in range(3):
            for g in range(nkv):
                ref = evict_ref(w[l, s, g].cpu(), lens[s], keep, first, recent)
                assert kept_c[l, s, g, :len(ref)].tolist() == ref
                hist[l][s][g] = ([hist[l][s][g][0][j] for j in ref], [hist[l][s][g][1][j] for j in ref])
                wref[l][s][g] = [wref[l][s][g][j] for j in ref]
    lens = new_len.tolist()
    w2 = torch.zeros((layers, 3, nkv, 4 * PAGE), device="cuda:0")
    w2[..., :keep] = w_kept
    for new in ([1, 1, 1], [5, 1, 3]):
        lens = step(dst, lens, new, w2)
