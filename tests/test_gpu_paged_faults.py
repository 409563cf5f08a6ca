"""Non-finite values and faulty lengths in the operators over caller-owned pages."""
import pytest

from test_gpu_paged_ops import PAGE, T

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
