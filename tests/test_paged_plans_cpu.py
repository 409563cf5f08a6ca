"""Host side of the operators over caller-owned K/V pages: how much scratch
they ask for, and refusals."""
import ctypes as C

import pytest

import vvq2

BASE = 1 << 20


def desc(**kw):
    d = dict(k=BASE, v=BASE, block_table=BASE, n_layers=2, n_pages=8, max_pages=1 << 16, n_seqs=3, n_kv_heads=2,
             head_dim=64, type=vvq2.F16)
    d.update(kw)
    return vvq2.PagesDesc(**d)


@pytest.mark.parametrize("n_seqs,nkv,nq,total,max_q,max_kv", [
    (48, 4, 20, 300_000, 12_000, 12_000), (160, 4, 28, 12_159, 12_000, 32_000), (65, 2, 14, 8064, 8000, 8000),
    (6, 2, 12, 9000, 4001, 4501), (1, 4, 28, 16_384, 16_384, 16_384), (1, 8, 8, 131_072, 131_072, 131_072),
    (1000, 8, 64, 1_000_000, 32_000, 100_000), (1, 1, 128, 4000, 4000, 4_000_000), (3, 1, 1, 2, 2, 64)])
def test_scratch_of_the_key_weights_is_bounded(n_seqs, nkv, nq, total, max_q, max_kv):
    d = desc(n_seqs=n_seqs, n_kv_heads=nkv)
    n = vvq2.lib().vvq2_attention_key_weights_workspace(C.addressof(d), total, max_q, max_kv, nq)
    assert n <= 32 << 20


def test_a_prompt_of_many_rows_asks_for_scratch():
    d = desc(n_seqs=1, n_kv_heads=4)
    assert vvq2.lib().vvq2_attention_key_weights_workspace(C.addressof(d), 8000, 8000, 8000, 28) > 0


def test_an_eviction_of_too_many_pages_is_refused_at_once():
    """More destination pages than a launch has blocks: an argument error, before anything runs."""
    d = desc(n_layers=1 << 10, n_seqs=1 << 10, n_kv_heads=8, max_pages=1 << 20)
    keep = 64 << 9
    rc = vvq2.lib().vvq2_pages_evict(C.addressof(d), 1 << 50, 1 << 9, 3 * BASE, keep, 1 << 51, keep, keep, 0, 0,
                                     1 << 52, None, 7 * BASE, None, None)
    assert rc == -2 and b"pages" in vvq2.lib().vvq2_last_error()
