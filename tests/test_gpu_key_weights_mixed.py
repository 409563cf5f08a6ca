"""Key weights of a packed batch of few long chunks and many single rows: the
long ones' rows are cut into chunks, the others' are not."""
import pytest

from test_gpu_paged_ops import Chunk, T, check_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dtype", [((14, 2, 64), "float16"), ((28, 4, 128), "bfloat16"),
                                         ((128, 1, 64), "float16")], ids=["64", "128", "one"])
@pytest.mark.parametrize("seqs", [[(1, 30 + 29 * s) for s in range(40)] + [(1200, 1200)] + [(0, 70), (5, 5), (1, 0)],
                                  [(900, 1500)] + [(2, 300 + s) for s in range(35)] + [(700, 700), (300, 2000)]],
                         ids=["single", "several"])
def test_long_chunks_among_single_rows(vv, heads, dtype, seqs):
    torch = T()
    c = Chunk(seqs, heads, getattr(torch, dtype), seed=61, pad=7).gpu()
    out, lse = c.attend()
    c.check(out, lse)
    shape = (len(seqs), c.nkv, c.max_kv + 3)
    prior, w_in = torch.randn(shape, device="cuda:0"), torch.rand(shape, device="cuda:0")
    got = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv, w_in=w_in, w_out=prior.clone())
    check_weights(c, lse, got, w_in, prior)
    for _ in range(3):
        again = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv, w_in=w_in,
                                         w_out=prior.clone())
        assert torch.equal(again, got)
    lib, p = vv.lib(), c.pages._p
    need = lib.vvq2_attention_key_weights_workspace(p, c.total, c.max_q, c.max_kv, c.nq)
    assert need > 0
    for n in (0, need // 5 // 16 * 16, need // 2 // 16 * 16, need, 4 * need):
        ws = torch.empty(max(16, n), dtype=torch.uint8, device="cuda:0")
        held = prior.clone()
        rc = lib.vvq2_attention_key_weights(p, 0, c.qd.data_ptr(), c.nq * c.hd, lse.data_ptr(), c.qs.data_ptr(),
                                            c.kl.data_ptr(), c.total, c.max_q, c.max_kv, c.nq, c.scale,
                                            w_in.data_ptr(), held.data_ptr(), held.shape[2],
                                            ws.data_ptr() if n else None, n, None,
                                            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        check_weights(c, lse, held, w_in, prior)


def test_a_slice_of_a_batch(vv):
    """Sequences whose rows begin inside q, with rows of others before and behind."""
    torch = T()
    c = Chunk([(70, 100), (600, 900), (1, 500), (400, 400), (3, 40)], (12, 2, 128), torch.float16, seed=62, pad=2).gpu()
    _, lse = c.attend()
    whole = vv.attention_key_weights(c.qd, lse, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    check_weights(c, lse, whole, None)
    pages = vv.Pages(c.pages.k, c.pages.v, c.pages.block_table[1:4].contiguous())
    lse[:70] = lse[-5:] = float("nan")
    part = vv.attention_key_weights(c.qd, lse, pages, c.qs[1:5].clone(), c.kl[1:4].clone(), c.max_q, c.max_kv)
    for s in range(3):
        kv = c.seqs[s + 1][1]
        assert torch.allclose(part[s, :, :kv], whole[s + 1, :, :kv], rtol=1e-5, atol=1e-30)
