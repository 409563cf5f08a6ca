"""Refusals of the operators over caller-owned K/V pages that need no GPU:
every argument the library can check by itself is an argument error (-2)
before any device is looked for, and well-formed calls without an sm_100
device fail instead of falling back."""
import ctypes as C

import pytest

import vvq2

BASE = 1 << 20          # never dereferenced: checks come first


def desc(**kw):
    d = dict(k=BASE, v=BASE, block_table=BASE, n_layers=2, n_pages=8, max_pages=4, n_seqs=3, n_kv_heads=2,
             head_dim=64, type=vvq2.F16)
    d.update(kw)
    return vvq2.PagesDesc(**d)


def attend(d=None, **kw):
    a = dict(layer=0, q=BASE, q_stride=14 * 64, q_start=BASE, kv_len=BASE, total_q=5, max_q=4, max_kv=100,
             n_heads=14, scale=0.125, out=BASE, out_stride=14 * 64, lse=None, ws=None, ws_n=0, err=None, stream=None)
    a.update(kw)
    d = desc() if d is None else d
    return vvq2.lib().vvq2_attention_paged(C.addressof(d), *a.values())


def weigh(d=None, **kw):
    a = dict(layer=0, q=BASE, q_stride=14 * 64, lse=BASE, q_start=BASE, kv_len=BASE, total_q=5, max_q=4, max_kv=100,
             n_heads=14, scale=0.125, w_in=None, w_out=BASE, w_stride=100, ws=None, ws_n=0, err=None, stream=None)
    a.update(kw)
    d = desc() if d is None else d
    return vvq2.lib().vvq2_attention_key_weights(C.addressof(d), *a.values())


def evict(d=None, **kw):
    a = dict(dst=2 * BASE, dst_max_pages=2, kv_len=3 * BASE, max_kv=200, w=4 * BASE, w_stride=200, keep=70, first=10,
             recent=60, kept=5 * BASE, w_out=6 * BASE, new_len=7 * BASE, err=None, stream=None)
    a.update(kw)
    d = desc() if d is None else d
    return vvq2.lib().vvq2_pages_evict(C.addressof(d), *a.values())


BAD_PAGES = [dict(k=None), dict(v=None), dict(block_table=None), dict(n_layers=0), dict(n_pages=0),
             dict(max_pages=0), dict(n_seqs=0), dict(n_kv_heads=0), dict(head_dim=32), dict(head_dim=96),
             dict(head_dim=256), dict(type=vvq2.F32), dict(type=vvq2.Q8_0), dict(k=BASE + 8), dict(v=BASE + 2),
             dict(block_table=BASE + 2), dict(n_pages=1 << 29), dict(n_pages=-1), dict(n_seqs=-5)]


@pytest.mark.parametrize("kw", BAD_PAGES, ids=lambda k: "-".join(f"{n}={v}" for n, v in k.items()))
def test_bad_pages_are_refused(kw):
    assert attend(desc(**kw)) == -2
    assert evict(desc(**kw)) == -2
    if "v" not in kw or kw["v"] is not None:
        assert weigh(desc(**kw)) == -2
    assert vvq2.lib().vvq2_attention_paged_workspace(C.addressof(desc(**kw)), 5, 4, 100, 14) == 0


ROWS = [dict(layer=2), dict(layer=-1), dict(q=None), dict(q_start=None), dict(kv_len=None), dict(total_q=-1),
        dict(max_q=-1), dict(max_q=0), dict(max_kv=-1), dict(n_heads=0), dict(n_heads=13), dict(n_heads=258),
        dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
        dict(q_stride=13 * 64), dict(q_stride=14 * 64 + 4), dict(q=BASE + 8), dict(q_start=BASE + 1),
        dict(kv_len=BASE + 3), dict(total_q=1 << 30, n_heads=14)]


@pytest.mark.parametrize("kw", ROWS, ids=lambda k: "-".join(f"{n}={v}" for n, v in k.items()))
def test_bad_chunks_are_refused(kw):
    assert attend(**kw) == -2
    assert weigh(**kw) == -2


@pytest.mark.parametrize("kw", [dict(out=None), dict(out=BASE + 8), dict(out_stride=13 * 64),
                                dict(out_stride=14 * 64 + 1), dict(lse=BASE + 2), dict(ws=BASE + 4, ws_n=64),
                                dict(err=BASE + 1)])
def test_attention_refusals(kw):
    assert attend(**kw) == -2


@pytest.mark.parametrize("kw", [dict(lse=None), dict(w_out=None), dict(w_stride=99), dict(w_stride=1 << 31),
                                dict(w_in=BASE + 4), dict(w_in=BASE + 2), dict(w_out=BASE + 2), dict(lse=BASE + 1),
                                dict(ws=BASE + 8, ws_n=64)])
def test_weight_refusals(kw):
    assert weigh(**kw) == -2


@pytest.mark.parametrize("kw", [dict(dst=None), dict(kv_len=None), dict(w=None), dict(kept=None), dict(new_len=None),
                                dict(max_kv=0), dict(w_stride=199), dict(keep=0), dict(keep=-3), dict(first=-1),
                                dict(recent=-1), dict(first=11), dict(first=71, recent=0), dict(dst_max_pages=1),
                                dict(dst_max_pages=0), dict(dst=BASE), dict(new_len=3 * BASE + 8),
                                dict(w_out=4 * BASE), dict(kept=4 * BASE + 64), dict(kept=6 * BASE),
                                dict(w=4 * BASE + 1)])
def test_evict_refusals(kw):
    assert evict(**kw) == -2


def test_null_descriptor():
    lib = vvq2.lib()
    z = [0] * 20
    assert lib.vvq2_attention_paged(None, 0, None, 0, None, None, 0, 0, 0, 0, 1.0, None, 0, None, None, 0, None,
                                    None) == -2
    assert lib.vvq2_attention_key_weights(None, 0, None, 0, None, None, None, 0, 0, 0, 0, 1.0, None, None, 0, None,
                                          0, None, None) == -2
    assert lib.vvq2_attention_key_weights_workspace(None, 1, 1, 1, 1) == 0
    assert lib.vvq2_pages_evict(None, None, *z[:1], None, 0, None, 0, 0, 0, 0, None, None, None, None, None) == -2
    assert lib.vvq2_last_error() == b"null pages"


def test_well_formed_calls_need_a_device():
    if vvq2.lib().vvq2_device_count() > 0:
        pytest.skip("a GPU is present")
    assert attend() in (-10, -9)
    assert weigh() in (-10, -9)
    assert evict() in (-10, -9)
    assert vvq2.lib().vvq2_attention_paged_workspace(C.addressof(desc()), 5, 4, 100, 14) == 0


def test_nothing_to_do_is_no_error():
    assert attend(total_q=0, max_q=0) == 0
    assert weigh(max_kv=0) == 0


def test_binding_checks_tensors():
    import torch
    k = torch.zeros((4, 2, 64, 64), dtype=torch.float16)
    bt = torch.zeros((1, 2), dtype=torch.int32)
    pages = vvq2.Pages(k, k.clone(), bt)
    assert (pages.n_layers, pages.n_pages, pages.n_kv, pages.head_dim) == (1, 4, 2, 64)
    for kk, vv, tt in [(k.float(), k, bt), (k, k.bfloat16(), bt), (k[:, :, :32], k[:, :, :32], bt),
                       (k, k[:3], bt), (k.transpose(0, 1), k.transpose(0, 1), bt), (k, k, bt.long()), (k, k, bt[0])]:
        with pytest.raises(vvq2.VVQ2Error):
            vvq2.Pages(kk, vv, tt)
    q = torch.zeros((3, 14, 64), dtype=torch.float16)
    qs, kl = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([9], dtype=torch.int32)
    for a in [(q.float(), qs, kl), (q[:, :, :32], qs, kl), (q.transpose(0, 1), qs, kl), (q, qs[:1], kl),
              (q, qs.long(), kl), (q, qs, kl.long()), (q, qs, torch.zeros(2, dtype=torch.int32))]:
        with pytest.raises(vvq2.VVQ2Error):
            vvq2._rows(pages, *a)
    assert vvq2._rows(pages, q, qs, kl) == (3, 14, 14 * 64)
    fused = torch.zeros((3, 18, 64), dtype=torch.float16)
    assert vvq2._rows(pages, fused[:, :14], qs, kl) == (3, 14, 18 * 64)
