"""Non-finite values and faulty lengths in the operators over caller-owned
pages, where several items share a block, and a tile has columns to spare."""
import math

import pytest

from test_gpu_paged_ops import PAGE, SMALL, Chunk, T

pytestmark = pytest.mark.gpu


def test_nonfinite_values_stay_in_their_item(vv):
    """Far more items than a block can number in 8 bits, each with a non-finite
    V element in one column of its last key: that column of the last row, and
    nothing else, is non-finite."""
    torch = T()
    n_seqs, nkv, hd, n_pages = 1100, 64, 64, 48       # 70,400 items: more than 256 in a block
    rng = torch.Generator(device="cuda:0").manual_seed(51)
    d = dict(device="cuda:0", generator=rng)
    k = torch.randn((n_pages, nkv, PAGE, hd), **d).half()
    v = torch.randn((n_pages, nkv, PAGE, hd), **d).half()
    col = torch.randint(0, hd, (n_pages, nkv), **d)
    v[:, :, 1].scatter_(2, col[..., None], float("inf"))
    page = torch.randint(0, n_pages, (n_seqs, 1), **d).int()
    q = torch.randn((2 * n_seqs, nkv, hd), **d).half()
    qs = (2 * torch.arange(n_seqs + 1, device="cuda:0")).int()
    kl = torch.full((n_seqs,), 2, dtype=torch.int32, device="cuda:0")
    out = vv.attention_paged(q, vv.Pages(k, v, page), qs, kl, 40, 64)       # (max_q x heads: not the few-row kernel)
    bad = ~torch.isfinite(out.view(n_seqs, 2, nkv, hd))
    assert not bad[:, 0].any()
    want = torch.zeros((n_pages, nkv, hd), dtype=torch.bool, device="cuda:0").scatter_(2, col[..., None], True)
    assert torch.equal(bad[:, 1], want[page[:, 0].long()])


@pytest.mark.parametrize("starts,lens", [([0, 40, 120, 130], [300, 200, 90]),      # the last starts past the rows
                                         ([0, 50, 40, 90], [300, 200, 90]),        # descending
                                         ([0, 40, 120, 120], [300, 200, 5000]),    # a length, of no new tokens
                                         ([0, 40, 120, 120], [300, 200, -1]),
                                         ([-3, 0, 120, 120], [0, 200, 9])])        # rows before the first
def test_every_clamped_length_sets_the_error_word(vv, starts, lens):
    torch = T()
    c = Chunk([(40, 300), (80, 200), (0, 90)], (14, 2, 64), torch.float16, seed=52).gpu()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda:0")
    _, lse = c.attend()
    for weigh in (False, True):
        err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
        # (5000 is cut to 300 keys, whose pages the table does not name either:
        # the weights read them, and of two words the later one stays)
        both = (5, 6) if weigh and lens[2] == 5000 else (5,)
        for qs, kl, words in ((c.qs, c.kl, (0,)), (i32(starts), i32(lens), both)):
            if weigh:
                vv.attention_key_weights(c.qd, lse, c.pages, qs, kl, 80, 300, err=err)
            else:
                vv.attention_paged(c.qd, c.pages, qs, kl, 80, 300, err=err)
            assert err.item() in words, weigh


@pytest.mark.parametrize("n", [1, 30], ids=["few", "many"])
@pytest.mark.parametrize("bad", [0, 40, 69])
def test_a_clamped_length_among_many_sequences(vv, bad, n):
    """No block meets all sequences on the way to its items."""
    torch = T()
    c = Chunk([(n, 100)] * 70, (14, 2, 64), torch.float16, seed=54).gpu()
    _, lse = c.attend()
    for weigh in (False, True):
        err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
        for length, word in ((100, 0), (101, 5)):
            c.kl[bad] = length
            if weigh:
                vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, 100, err=err)
            else:
                vv.attention_paged(c.qd, c.pages, c.qs, c.kl, c.max_q, 100, err=err)
            assert err.item() == word, (weigh, length)
        c.kl[bad] = 100


@pytest.mark.parametrize("heads", [(14, 2, 64), (9, 3, 128), (6, 1, 64), (4, 4, 64)],
                         ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("n", [1, 3, 18, 200])
def test_a_key_of_minus_infinite_scores_has_no_weight(vv, heads, n):
    """A visible key with an element of -inf that every query multiplies by a
    positive one has scores of -inf: weight 0, and the other keys have theirs.
    (Group sizes whose rows do not fill the columns of a tile among them.)"""
    torch = T()
    kv, j = n + 300, 10
    c = Chunk([(n, kv), (2, 40)], heads, torch.float16, seed=53)
    c.q[..., 0] = c.q[..., 0].abs() + 0.5
    zeroed = c.keys[0].clone()
    zeroed[j] = 0
    c.K[c.bt[0, 0], :, j, 0] = float("-inf")
    c.gpu()
    _, lse = c.attend()
    assert torch.isfinite(lse).all()
    w = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    for g in range(c.nkv):
        hs = slice(g * c.G, (g + 1) * c.G)
        q, K = c.q[:n, hs].double().cuda(), zeroed[:, g].double().cuda()
        x = torch.einsum("thd,jd->thj", q, K) * c.scale
        E = c.hd * 2.0 ** -23 * c.scale * torch.einsum("thd,jd->thj", q.abs(), K.abs())
        hide = (torch.arange(kv)[None, :] >= (kv - n + torch.arange(n) + 1)[:, None]).cuda()
        hide[:, j] = True
        x = x.masked_fill(hide[:, None], -math.inf)
        l = lse[:n, hs].double()[..., None]
        assert ((torch.logsumexp(x, -1, keepdim=True) - l).abs() <=
                E.amax(-1, keepdim=True) + SMALL + kv * 2.0 ** -22 + l.abs() * 2.0 ** -22).all()
        p = torch.exp(x - l)
        want = p.sum((0, 1))
        tol = ((E + SMALL + l.abs() * 2.0 ** -22) * p).sum((0, 1)) + want * (n * c.G + 8) * 2.0 ** -23 + 1e-30
        assert ((w[0, g, :kv].double() - want).abs() <= tol).all(), (g, w[0, g, j].item())
