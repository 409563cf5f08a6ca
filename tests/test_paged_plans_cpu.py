"""Host side of the operators over caller-owned K/V pages: how much scratch
they ask for, what the binding keeps of a failed call, and refusals."""
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


class FakeLib:
    """Entry points of the library that note what they get."""

    def __init__(self):
        self.query, self.rc, self.scratch = 0, -9, []

    def vvq2_attention_paged_workspace(self, *a):
        return self.query

    vvq2_attention_key_weights_workspace = vvq2_attention_paged_workspace

    def vvq2_attention_paged(self, *a):
        self.scratch.append(a[15])
        return self.rc

    def vvq2_attention_key_weights(self, *a):
        self.scratch.append(a[16])
        return self.rc

    def vvq2_last_error(self):
        return b"no device"


@pytest.fixture
def fake(monkeypatch):
    f = FakeLib()
    monkeypatch.setattr(vvq2, "_lib", f)
    monkeypatch.setattr(vvq2, "lib", lambda: f)
    monkeypatch.setattr(vvq2, "_current_stream", lambda device: 0)
    return f


def tensors():
    import torch
    k = torch.zeros((4, 2, 64, 64), dtype=torch.float16)
    pages = vvq2.Pages(k, k.clone(), torch.zeros((1, 2), dtype=torch.int32))
    q = torch.zeros((3, 14, 64), dtype=torch.float16)
    return q, pages, torch.tensor([0, 3], dtype=torch.int32), torch.tensor([9], dtype=torch.int32)


@pytest.mark.parametrize("op", ["attend", "weigh"])
def test_a_failed_query_of_scratch_is_not_kept(fake, op):
    import torch
    q, pages, qs, kl = tensors()
    lse = torch.zeros((3, 14))

    def call():
        if op == "attend":
            return vvq2.attention_paged(q, pages, qs, kl, 3, 9)
        return vvq2.attention_key_weights(q, lse, pages, qs, kl, 3, 9)

    with pytest.raises(vvq2.VVQ2Error):
        call()
    fake.query, fake.rc = 640, 0
    call()
    fake.query = 0            # a size that served a call is kept
    call()
    assert fake.scratch == [0, 640, 640]


def test_tensors_that_require_grad_are_refused(fake):
    """The operators have no backward: a result that is silently detached would be wrong."""
    import torch
    fake.rc = 0
    q, pages, qs, kl = tensors()
    lse, w = torch.zeros((3, 14)), torch.zeros((1, 2, 9))
    dst = torch.ones((1, 2), dtype=torch.int32)
    fake.vvq2_pages_evict = lambda *a: 0
    calls = {"attend": lambda: vvq2.attention_paged(q, pages, qs, kl, 3, 9),
             "weigh": lambda: vvq2.attention_key_weights(q, lse, pages, qs, kl, 3, 9, w_in=w, w_out=w.clone()),
             "evict": lambda: vvq2.pages_evict(pages, dst, kl, w, 4)}
    takes = {"attend": [q, pages.k, pages.v], "weigh": [q, lse, pages.k, w], "evict": [pages.k, pages.v, w]}
    for name, call in calls.items():
        call()
        for t in takes[name]:
            t.requires_grad_(True)
            with pytest.raises(vvq2.VVQ2Error) as e:
                call()
            assert e.value.rc == -2 and "grad" in str(e.value)
            with torch.no_grad():
                call()
            t.requires_grad_(False)
        call()
