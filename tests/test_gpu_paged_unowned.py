"""Rows that no sequence owns, around the rows of vvq2_attention_paged: those
before q_start[0] (a slice of a packed batch), padding behind the last
sequence, and rows past max_q.  Their outputs keep every bit, whether the keys
are split over the GPU or not."""
import pytest

from test_gpu_paged_ops import PAGE, Chunk, T

pytestmark = pytest.mark.gpu

# (new tokens, cached keys) of a packed batch, of which the call gets the
# sequences from the second on: for the few-row kernel, for the 128-row one
# with a tile per sequence, and with several
BATCHES = {"few": [(5, 90), (1, 3000), (0, 10), (2, 2500), (1, 70)],
           "tile": [(30, 50), (9, 700), (7, 3000), (0, 0), (12, 2100)],
           "tiles": [(50, 60), (40, 700), (7, 3000), (0, 3), (90, 1100)]}
HEADS = [(14, 2, 64), (28, 4, 128)]


def later(vv, c):
    """The batch without its first sequence."""
    return vv.Pages(c.pages.k, c.pages.v, c.pages.block_table[1:].contiguous()), c.qs[1:].clone(), c.kl[1:].clone()


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in_place"])
@pytest.mark.parametrize("heads", HEADS, ids=["64", "128"])
@pytest.mark.parametrize("batch", BATCHES)
def test_rows_of_no_sequence_keep_their_outputs(vv, batch, heads, in_place):
    torch = T()
    c = Chunk(BATCHES[batch], heads, torch.float16, seed=41, pad=3).gpu()
    pages, qs, kl = later(vv, c)
    first, last = c.starts[1], c.starts[-1]
    max_q = max(n for n, _ in c.seqs[1:])
    out = c.qd.clone() if in_place else torch.full_like(c.qd, 5.0)
    lse = torch.full((c.total, c.nq), 9.0, device="cuda:0")
    before = out.clone()
    err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    q = out if in_place else c.qd
    assert vv.lib().vvq2_attention_paged_workspace(pages._p, c.total, max_q, c.max_kv, c.nq) > 0   # keys are split
    vv.attention_paged(q, pages, qs, kl, max_q, c.max_kv, out=out, lse=lse, err=err)
    assert err.item() == 0
    assert torch.equal(out[:first], before[:first]) and (lse[:first] == 9).all()
    assert torch.equal(out[last:], before[last:]) and (lse[last:] == 9).all()
    ref, tol, rl, ltol = c.reference()
    own = slice(first, last)
    assert ((out[own].double() - ref[own]).abs() <= tol[own]).all()
    none = torch.isinf(rl[own])
    assert torch.equal(torch.isneginf(lse[own]), none)
    assert ((lse[own].double() - rl[own]).abs() <= ltol[own])[~none].all()


@pytest.mark.parametrize("heads", HEADS, ids=["64", "128"])
@pytest.mark.parametrize("seqs,max_q", [([(6, 3000), (2, 2500)], 2), ([(20, 3000), (3, 500)], 8),
                                        ([(70, 3000), (3, 500)], 40)], ids=["few", "tile", "tiles"])
def test_rows_past_max_q_keep_their_outputs(vv, seqs, max_q, heads):
    torch = T()
    c = Chunk(seqs, heads, torch.bfloat16, seed=42, pad=2).gpu()
    out, lse = torch.full_like(c.qd, 5.0), torch.full((c.total, c.nq), 9.0, device="cuda:0")
    err = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    vv.attention_paged(c.qd, c.pages, c.qs, c.kl, max_q, c.max_kv, out=out, lse=lse, err=err)
    assert err.item() == 5
    cut = slice(max_q, c.starts[1])
    assert (out[cut] == 5).all() and (lse[cut] == 9).all()
    assert (out[c.starts[-1]:] == 5).all() and (lse[c.starts[-1]:] == 9).all()
    # the other sequence has all its rows
    ref, tol, rl, ltol = c.reference()
    own = slice(c.starts[1], c.starts[2])
    assert ((out[own].double() - ref[own]).abs() <= tol[own]).all()
    assert ((lse[own].double() - rl[own]).abs() <= ltol[own]).all()


def test_scratch_follows_the_rows_of_the_sequences(vv):
    """One decode row of a large packed batch asks for no more than alone."""
    torch = T()
    c = Chunk([(3, 30), (1, 5000)], (28, 4, 128), torch.float16, seed=43, pad=3000).gpu()
    pages, qs, kl = later(vv, c)
    size = lambda rows: vv.lib().vvq2_attention_paged_workspace(pages._p, rows, 1, 5000, 28)
    assert 0 < size(1) == size(c.total) == size(100_000)
    out, lse = torch.full_like(c.qd, 5.0), torch.full((c.total, c.nq), 9.0, device="cuda:0")
    vv.attention_paged(c.qd, pages, qs, kl, 1, 5000, out=out, lse=lse)
    ref, tol, rl, ltol = c.reference()
    assert ((out[3:4].double() - ref[3:4]).abs() <= tol[3:4]).all()
    assert ((lse[3:4].double() - rl[3:4]).abs() <= ltol[3:4]).all()
    assert (out[:3] == 5).all() and (out[4:] == 5).all() and (lse[:3] == 9).all() and (lse[4:] == 9).all()
    alone = vv.attention_paged(c.qd[3:4], pages, qs - 3, kl, 1, 5000)
    assert torch.equal(alone, out[3:4])


@pytest.mark.parametrize("n_seqs", [31, 32, 33, 64, 65, 1030])
def test_few_rows_among_many_sequences(vv, n_seqs):
    """Split keys in a batch of mostly empty sequences: a row's sequence is found among them all."""
    torch = T()
    seqs = [(0, 3)] * n_seqs
    rows = {0: (41, 300), 1: (2, 2100), n_seqs // 2: (5, 1500), n_seqs - 2: (1, 90), n_seqs - 1: (50, 60)}
    for s, x in rows.items():
        seqs[s] = x
    c = Chunk(seqs, (14, 2, 64), torch.float16, seed=44, pad=2).gpu()
    assert vv.lib().vvq2_attention_paged_workspace(c.pages._p, c.total, c.max_q, c.max_kv, c.nq) > 0
    out, lse = torch.full_like(c.qd, 5.0), torch.full((c.total, c.nq), 9.0, device="cuda:0")
    vv.attention_paged(c.qd, c.pages, c.qs, c.kl, c.max_q, c.max_kv, out=out, lse=lse)
    c.check(out, lse)
    assert (out[-2:] == 5).all() and (lse[-2:] == 9).all()
