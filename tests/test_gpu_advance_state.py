"""The state after the accepted tokens of a step (``ops.advance_state``) against the recurrence in 64 bits.

Bounds: a WKV step multiplies and adds with fp32 roundings (2^-24 each) and exponentials of fp32 arguments; the arguments are sums of up to
n decays and a key, each rounded (2^-24 of their magnitude, which the running maximum and the decays bound), so after n steps a sum is off by at most
n * (8 + |largest argument|) * 2^-23 of the sum of its terms' magnitudes.  A layer norm sums C values in partial sums of at most C / 1024 + 13 additions and
then subtracts, divides, multiplies and adds: (C / 1024 + 24) * 2^-23 of the larger of its terms."""
import pytest
import torch

from rwkvstic_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(B, L, T, C, seed=0):
    g = torch.Generator().manual_seed(seed)
    state = torch.randn(B, L, 5, C, generator=g)
    state[:, :, 3] = 1 + 9 * torch.rand(B, L, C, generator=g)
    trace = torch.randn(L, 4, B, T, C, generator=g)
    trace[:, :2] = trace[:, :2] * 2 + 0.5
    params = torch.randn(L, 5, C, generator=g)
    params[:, 4] = -torch.exp(torch.rand(L, C, generator=g) * 8 - 5)
    counts = torch.randint(0, T + 1, (B,), generator=g)
    return state.to(DEV), counts.to(DEV), trace.to(DEV), params.to(DEV)


def check(state, counts, trace, params, out=None):
    B, L, _, C = state.shape
    T = trace.shape[3]
    want, size, far = state.double().cpu(), state.double().abs().cpu(), state[:, :, 4].double().abs().cpu()
    tr, pr = trace.double().cpu(), params.double().cpu()
    moved = torch.zeros(B, dtype=torch.bool)
    for b, n in enumerate(counts.tolist()):
        n = min(max(n, 0), T)
        moved[b] = n > 0
        for t in range(n):
            for row in (0, 1):
                x = tr[:, row, b, t]
                d = x - x.mean(-1, keepdim=True)
                s = (d.square().mean(-1, keepdim=True) + 1e-5).sqrt()
                want[b, :, row] = d / s * pr[:, 2 * row] + pr[:, 2 * row + 1]
                # terms: x and its mean over the deviation, times the weight, and the bias
                size[b, :, row] = ((x.abs() + x.mean(-1, keepdim=True).abs()) / s * pr[:, 2 * row].abs() + pr[:, 2 * row + 1].abs()) * (C / 1024 + 24)
            k, v, w = tr[:, 2, b, t], tr[:, 3, b, t], pr[:, 4]
            p = torch.maximum(want[b, :, 4] + w, k)
            f, e = torch.exp(want[b, :, 4] + w - p), torch.exp(k - p)
            want[b, :, 2], want[b, :, 3] = f * want[b, :, 2] + e * v, f * want[b, :, 3] + e
            size[b, :, 2], size[b, :, 3] = f * size[b, :, 2] + e * v.abs(), f * size[b, :, 3] + e
            far[b] = far[b] + w.abs() + k.abs()
            want[b, :, 4] = p
        size[b, :, 2:4] *= (n + 1) * (8 + far[b].unsqueeze(1))
        size[b, :, 4] = (n + 1) * far[b]
    before = state.clone()
    got = ops.advance_state(state, counts, trace, params, out)
    torch.cuda.synchronize()
    assert got is (state if out is None else out)
    if out is not None:
        assert torch.equal(state, before)
    assert torch.equal(got.cpu()[~moved], before.cpu()[~moved])
    err = (got.double().cpu() - want).abs() - size * 2.0 ** -23
    assert float(err.max()) <= 0.0, [float(err[:, :, i].max()) for i in range(5)]


@pytest.mark.parametrize("B,L,T,C", [(1, 1, 1, 4), (1, 12, 5, 768), (7, 3, 4, 128), (3, 2, 9, 1028), (2, 1, 40, 1536), (33, 2, 2, 20), (2, 2, 3, 5120), (130, 1, 1, 64)])
def test_against_recurrence(B, L, T, C):
    args = make(B, L, T, C, seed=B)
    check(*args, out=torch.full_like(args[0], 3.0))
    check(*args)


def test_counts_are_clamped_and_the_rest_of_a_trace_is_not_read():
    state, _, trace, params = make(5, 2, 3, 64)
    counts = torch.tensor([-3, 0, 2, 3, 2 ** 40], device=DEV)
    trace[:, :, 0] = trace[:, :, 1] = float("nan")
    trace[:, :, 2, 2:] = float("nan")
    check(state, counts, trace, params, torch.empty_like(state))
    check(state, counts, trace, params)


def test_empty_state_and_a_decay_that_forgets_at_once():
    state, counts, trace, params = make(4, 2, 6, 128)
    counts.fill_(6)
    state.zero_()
    state[:, :, 4] = -1e30
    w = params[:, 4].clone()
    got = ops.advance_state(state, counts, trace, params, torch.empty_like(state))
    assert torch.isfinite(got).all()
    # from an empty state the sums are those of the tokens alone, whatever stood in front
    y = torch.zeros(4, 6, 128, device=DEV)
    aa, bb, pp = (state[:, 0, i].contiguous() for i in (2, 3, 4))
    ops.wkv_scan(w[0].contiguous(), torch.zeros(128, device=DEV), trace[0, 2].contiguous(), trace[0, 3].contiguous(), aa, bb, pp)
    # six steps with arguments up to 6 * 20 in magnitude: 6 * 128 * 2^-23 of a sum of terms, and |value| < 5
    assert ((got[:, 0, 2] - aa).abs() <= 5e-4 * bb).all() and ((got[:, 0, 3] - bb).abs() <= 1e-4 * bb).all()
    assert ((got[:, 0, 4] - pp).abs() <= 1e-5 * (1 + pp.abs())).all()
    params[:, 4] = -float("inf")
    got = ops.advance_state(state, counts, trace, params, torch.empty_like(state))
    assert torch.equal(got[:, :, 2], trace[:, 3, :, 5].transpose(0, 1)) and torch.equal(got[:, :, 4], trace[:, 2, :, 5].transpose(0, 1))
    assert torch.equal(got[:, :, 3], torch.ones_like(got[:, :, 3]))


def test_a_stream_does_not_depend_on_the_other_streams():
    state, counts, trace, params = make(20, 3, 5, 256, seed=2)
    got = ops.advance_state(state, counts, trace, params, torch.empty_like(state))
    for b in (0, 7, 19):
        one = ops.advance_state(state[b:b + 1].contiguous(), counts[b:b + 1], trace[:, :, b:b + 1].contiguous(), params)
        assert torch.equal(one[0], got[b])


def test_captured_call_follows_its_counts():
    state, counts, trace, params = make(6, 2, 4, 128, seed=5)
    out = torch.empty_like(state)
    ops.advance_state(state, counts, trace, params, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.advance_state(state, counts, trace, params, out)
    for seed in range(3):
        counts.copy_(torch.randint(0, 5, (6,), generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.advance_state(state, counts, trace, params, torch.empty_like(state)))


def test_refusals():
    state, counts, trace, params = make(3, 2, 4, 64)
    for args in [(state.double(), counts, trace, params), (state[:, :1], counts, trace, params), (state, counts.int(), trace, params),
                 (state, counts[:2], trace, params), (state, counts, trace[:, :3], params), (state, counts, trace, params[:, :4]),
                 (state, counts, trace.transpose(2, 3), params), (state, counts, trace, params, state[:2]), (state.cpu(), counts, trace, params),
                 (state, counts.cpu(), trace, params), (state[0], counts, trace, params)]:
        with pytest.raises(ValueError):
            ops.advance_state(*args)
    with pytest.raises(_lib.B200RWKVError):
        ops.advance_state(torch.zeros(1, 1, 5, 6, device=DEV), counts[:1], torch.zeros(1, 4, 1, 2, 6, device=DEV), torch.zeros(1, 5, 6, device=DEV))
    same = state.clone()
    assert torch.equal(ops.advance_state(state, counts, trace[:, :, :, :0].contiguous(), params), same)
    assert ops.advance_state(state[:0], counts[:0], trace[:, :, :0].contiguous(), params).shape[0] == 0


def test_outputs_that_overlap_are_refused():
    state, counts, trace, params = make(3, 2, 4, 64)
    room = torch.zeros(4, 2, 5, 64, device=DEV)
    for bad in [(room[:3], counts, trace, params, room[1:]), (state, counts, trace, params, trace.view(-1)[:state.numel()].view_as(state))]:
        with pytest.raises(_lib.B200RWKVError, match="apart"):
            ops.advance_state(*bad)
    room[:3] = state
    again = ops.advance_state(room[:3], counts, trace, params, room[:3])       # the same memory under another name
    assert torch.equal(again, ops.advance_state(state, counts, trace, params, torch.empty_like(state)))
