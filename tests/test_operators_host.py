"""Refusals of the adapter, verification and state-advance entry points that need no GPU: codes and texts, no aborts."""
import ctypes as C

import pytest
import torch

from rwkvstic_b200 import _lib, ops

FAKE = 0x1000          # never dereferenced: every call below is refused before a launch


def adapt(nmat=1, n=2, rank=8, k=64, dtype=1, row_dtype=0, streams=2, tokens=3, a=FAKE, b=FAKE, x=FAKE, y=FAKE, out=FAKE, ids=FAKE, ws=FAKE,
          n_out=32, nbytes=0):
    banks = (_lib.Adapters * max(nmat, 1))(*[_lib.Adapters(a, b, None, n_out) for _ in range(max(nmat, 1))])
    p = lambda v: (C.c_void_p * max(nmat, 1))(*[v] * max(nmat, 1))
    return _lib.lib().b200rwkv_adapt_rows(nmat, banks, n, rank, k, dtype, p(x), p(y), p(out), row_dtype, ids, streams, tokens, ws, nbytes, None)


@pytest.mark.parametrize("change", [dict(nmat=0), dict(nmat=4), dict(n=0), dict(rank=0), dict(rank=6), dict(rank=260), dict(k=0), dict(k=12), dict(dtype=3),
                                    dict(row_dtype=2), dict(row_dtype=-1), dict(dtype=0, row_dtype=1), dict(streams=0), dict(tokens=0),
                                    dict(streams=65536, tokens=1), dict(streams=256, tokens=257), dict(n_out=0), dict(n_out=-5), dict(ids=None), dict(ws=None),
                                    dict(ws=0x1001)])
def test_adapt_rows_refuses(change):
    assert adapt(**change) == _lib.EINVAL
    assert b"adapt_rows" in _lib.lib().b200rwkv_last_error()


def test_adapt_rows_workspace_of_a_refused_size_is_zero():
    banks = (_lib.Adapters * 1)(_lib.Adapters(FAKE, FAKE, None, 32))
    L = _lib.lib()
    assert L.b200rwkv_adapt_rows_workspace_bytes(1, banks, 2, 6, 64, 1, 2, 3) == 0
    assert L.b200rwkv_adapt_rows_workspace_bytes(1, None, 2, 8, 64, 1, 2, 3) == 0
    assert L.b200rwkv_adapt_rows_workspace_bytes(1, banks, 2, 8, 64, 9, 2, 3) == 0


def verify(target=FAKE, draft=FAKE, tokens=FAKE, u=FAKE, lengths=None, streams=2, drafts=3, n=100, out=FAKE, accepted=FAKE, ws=FAKE, nbytes=1 << 30,
           ts=400, tr=100, ds=300, dr=100):
    return _lib.lib().b200rwkv_verify_drafts(target, ts, tr, draft, ds, dr, tokens, u, lengths, streams, drafts, n, out, accepted, ws, nbytes, None)


@pytest.mark.parametrize("change", [dict(target=None), dict(tokens=None), dict(u=None), dict(out=None), dict(accepted=None), dict(ws=None), dict(ws=0x1004),
                                    dict(nbytes=8), dict(streams=0), dict(streams=65536), dict(drafts=-1), dict(drafts=65), dict(n=0), dict(n=524289),
                                    dict(ts=-1), dict(tr=-1), dict(ds=-1), dict(dr=-1)])
def test_verify_drafts_refuses(change):
    assert verify(**change) == _lib.EINVAL
    assert b"verify_drafts" in _lib.lib().b200rwkv_last_error()


def test_verify_drafts_workspace():
    L = _lib.lib()
    assert L.b200rwkv_verify_drafts_workspace_bytes(4, 3, 1025) == 4 * 7 * 2 * 8
    assert L.b200rwkv_verify_drafts_workspace_bytes(0, 3, 10) == 0 and L.b200rwkv_verify_drafts_workspace_bytes(1, 65, 10) == 0


@pytest.mark.parametrize("change", [dict(state=None), dict(out=None), dict(counts=None), dict(trace=None), dict(params=None), dict(streams=0), dict(layers=0),
                                    dict(tokens=0), dict(channels=0), dict(channels=6), dict(state=0x1004), dict(out=0x1008), dict(trace=0x1001)])
def test_advance_state_refuses(change):
    args = {**dict(state=FAKE, out=FAKE, counts=FAKE, trace=FAKE, params=FAKE, streams=1, layers=2, tokens=3, channels=64), **change}
    assert _lib.lib().b200rwkv_advance_state(*args.values(), None) == _lib.EINVAL
    assert b"advance_state" in _lib.lib().b200rwkv_last_error()


def test_operators_need_cuda_tensors():
    z = torch.zeros
    with pytest.raises(RuntimeError):
        ops.adapt_rows([(z(1, 4, 8), z(1, 3, 4), None)], [z(2, 8)], z(1, dtype=torch.int64), [z(2, 3)])
    with pytest.raises(ValueError):
        ops.verify_drafts(z(1, 2, 5), None, z(1, 1, dtype=torch.int64), z(1, 2))
    with pytest.raises(ValueError):
        ops.advance_state(z(1, 1, 5, 4), z(1, dtype=torch.int64), z(1, 4, 1, 1, 4), z(1, 5, 4))


def test_pack_adapters():
    a, b, s = ops.pack_adapters([(torch.ones(3, 16), torch.ones(5, 3), 2.0), (torch.ones(6, 16), torch.ones(5, 6), 0.5)], torch.float16)
    assert a.shape == (2, 8, 16) and b.shape == (2, 5, 8) and s.tolist() == [2.0, 0.5] and a.dtype == b.dtype == torch.float16
    assert a.float().sum() == 16 * 9 and b.float().sum() == 5 * 9 and float(a[0, 3:].abs().sum()) == 0
    for bad in ([], [(torch.ones(3, 16), torch.ones(5, 4), 1.0)], [(torch.ones(3, 16), torch.ones(5, 3), 1.0), (torch.ones(3, 15), torch.ones(5, 3), 1.0)]):
        with pytest.raises(ValueError):
            ops.pack_adapters(bad)


@pytest.mark.skipif(torch.cuda.is_available(), reason="what a host without a device gets")
def test_adapt_rows_status_without_a_device():
    L = _lib.lib()
    assert L.b200rwkv_adapt_rows_status_word() is None
    assert L.b200rwkv_adapt_rows_status(None) == _lib.ECUDA and b"no CUDA device" in L.b200rwkv_last_error()


def test_adapt_rows_refuses_a_k_in_that_blocks_of_it_would_pass_32_bits():
    for k in (2 ** 31 - 8, 2 ** 30 + 8):
        assert adapt(k=k) == _lib.EINVAL and b"k_in" in _lib.lib().b200rwkv_last_error()
