"""Refusals of the paged cache's C entry points that need no GPU: every one of them returns before anything is launched."""
import ctypes as C

import pytest
import torch

from multimodal_amd import _lib as L

P = 1 << 20                                              # an aligned address that nothing reads


def _attn(**kw):
    a = L.PagedAttnArgs(q=P, k_new=P, v_new=P, kpool=P, vpool=2 * P, o=P, weights=None, page_table=P, lengths=P, positions=None, cos_t=P, sin_t=P,
                        B=2, H=4, Hkv=2, d=64, rot=32, page=16, n_pages=10, width=4, ld_table=4, ld_q=256, ld_k=128, ld_v=128, n_pos=64, mode=0, dtype=1,
                        workspace=P, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(a, k, v)
    return L.lib().mm_paged_decode_attn(C.byref(a), None)


@pytest.mark.parametrize("bad", [dict(kpool=None), dict(q=None), dict(o=None), dict(lengths=None), dict(page_table=None), dict(v_new=None), dict(kpool=P + 8),
                                 dict(H=3), dict(H=0), dict(Hkv=0), dict(d=66), dict(d=516), dict(d=0), dict(rot=31), dict(rot=66), dict(cos_t=None),
                                 dict(n_pos=0), dict(page=12), dict(page=2), dict(page=2048), dict(n_pages=0), dict(n_pages=1 << 31), dict(width=0),
                                 dict(width=1 << 28), dict(ld_table=-1), dict(ld_q=-1), dict(mode=2), dict(dtype=2), dict(B=-1), dict(B=65536)], ids=str)
def test_attend_refuses(bad):
    assert _attn(**bad) == -1 and b"paged_decode_attn" in L.lib().mm_last_error()


def test_attend_without_rows_does_nothing():
    assert _attn(B=0, q=None, o=None, lengths=None) == 0


@pytest.mark.parametrize("bad", [dict(k=None), dict(vpool=None), dict(S=-1), dict(S=1 << 30), dict(rot=1), dict(sin_t=None), dict(ld_k=-1), dict(bs_v=-1), dict(d=6),
                                 dict(dtype=7), dict(page=5)], ids=str)
def test_fill_refuses(bad):
    a = L.PagedFillArgs(k=P, v=P, kpool=P, vpool=2 * P, weights=None, page_table=P, start=None, counts=None, positions=None, cos_t=P, sin_t=P, B=2, S=3, Hkv=2, d=64,
                        rot=32, page=16, n_pages=10, width=4, ld_table=4, ld_k=128, bs_k=384, ld_v=128, bs_v=384, n_pos=64, dtype=1)
    for k, v in bad.items():
        setattr(a, k, v)
    assert L.lib().mm_paged_cache_fill(C.byref(a), None) == -1 and b"paged_cache_fill" in L.lib().mm_last_error()


@pytest.mark.parametrize("bad", [dict(budget=0), dict(recent=9), dict(recent=-1), dict(weights=None), dict(lengths=None), dict(kept=None), dict(workspace=None),
                                 dict(nbytes=0), dict(d=2), dict(page=6), dict(dtype=3)], ids=str)
def test_evict_refuses(bad):
    a = dict(kpool=P, vpool=2 * P, weights=P, table=P, lengths=P, kept=P, B=2, Hkv=2, d=64, page=16, n_pages=10, width=4, ld=4, budget=8, recent=2, dtype=1,
             workspace=P, nbytes=1 << 40, stream=None)
    a.update(bad)
    assert L.lib().mm_paged_evict(*a.values()) == -1 and b"paged_evict" in L.lib().mm_last_error()


@pytest.mark.parametrize("bad", [dict(p=None), dict(u=None), dict(tokens=None), dict(accepted=None), dict(drafts=None), dict(V=0), dict(K=-1), dict(B=-1), dict(ld_p=-1)],
                         ids=str)
def test_verify_refuses(bad):
    a = L.VerifyArgs(drafts=P, p=P, q=P, u=P, counts=None, tokens=P, accepted=P, B=2, K=3, V=50, ld_drafts=3, bs_p=200, ld_p=50, bs_q=150, ld_q=50, ld_u=4,
                     workspace=P, workspace_bytes=1 << 40)
    for k, v in bad.items():
        setattr(a, k, v)
    assert L.lib().mm_verify_drafts(C.byref(a), None) == -1 and b"verify_drafts" in L.lib().mm_last_error()


def test_null_arguments():
    for fn in ("mm_paged_decode_attn", "mm_paged_cache_fill", "mm_verify_drafts"):
        assert getattr(L.lib(), fn)(None, None) == -1


def test_wrappers_refuse_host_tensors():
    from multimodal_amd import ops
    pool, w, table, n = torch.zeros(3, 2, 16, 64), torch.zeros(3, 2, 16), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 128)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.paged_decode_attn(x, x, x, pool, pool.clone(), table, n, 2, 0, None, None, False)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.paged_cache_fill(x[:, None], x[:, None], pool, pool.clone(), table, 0, None, None)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.paged_evict(pool, pool.clone(), w, table, n, 4, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.verify_drafts(torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 2, 5), torch.zeros(2, 2))
