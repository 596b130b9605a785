"""Steps with drafted tokens through the whole model, and the operators of such a step run together as a server would."""
import numpy as np
import pytest
import torch

from rwkvstic_b200 import _lib, ops
from rwkvstic_b200.model import B200RWKV
from rwkvstic_b200.quant import quantize_fastquant
from rwkvstic_b200.synth import synth_checkpoint

from test_gpu_verify_drafts import rule

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
L, D, V = 3, 256, 515
TOL = 2e-3                 # max |dlogit|, as for the model's other paths


@pytest.fixture(scope="module")
def model():
    return B200RWKV.from_checkpoint(synth_checkpoint(L, D, vocab=V, seed=12), device=DEV)


def start(model, B, seed=0):
    """States in the middle of a text."""
    g = torch.Generator().manual_seed(seed)
    state = model.empty_batch_state(B)
    model.forward_rows(torch.randint(0, V, (B, 7), generator=g).to(DEV), state)
    return state, g


def close_states(a, b):
    """Carries are layer-normed rows, sums weighted values: fp32 through three blocks on two paths."""
    for row in range(5):
        scale = b[:, :, row].abs().max()
        assert float((a[:, :, row] - b[:, :, row]).abs().max()) <= 1e-4 * float(scale) + 1e-6, row


@pytest.mark.parametrize("B,T", [(1, 1), (1, 5), (6, 4), (40, 3), (3, 33)])
def test_draft_logits_are_those_of_every_prefix(model, B, T):
    state, g = start(model, B, seed=B)
    before = state.clone()
    tokens = torch.randint(0, V, (B, T), generator=g).to(DEV)
    logits, trace = model.forward_draft(tokens, state)
    assert tuple(logits.shape) == (B, T, V) and tuple(trace.shape) == (L, 4, B, T, D)
    assert torch.equal(state, before)
    model.check_rows_status()
    for t in range(T):
        s = before.clone()
        want = model.forward_rows(tokens[:, :t + 1], s)
        assert float((logits[:, t] - want).abs().max()) < TOL
        got = model.accept(before.clone(), trace, torch.full((B,), t + 1, device=DEV))
        close_states(got, s)


def test_streams_accept_different_numbers(model):
    B, T = 5, 4
    state, g = start(model, B)
    tokens = torch.randint(0, V, (B, T), generator=g).to(DEV)
    counts = torch.tensor([0, 1, 2, 3, 4], device=DEV)
    want = state.clone()
    for b in range(1, B):
        model.forward_rows(tokens[b:b + 1, :b], want[b:b + 1])
    _, trace = model.forward_draft(tokens, state)
    untouched = state[0].clone()
    assert model.accept(state, trace, counts) is state
    assert torch.equal(state[0], untouched)
    close_states(state, want)


def test_the_first_accept_may_be_a_captured_one():
    """What accept needs of the weights is there before it is called, so an eager call behind a capture has it too."""
    model = B200RWKV.from_checkpoint(synth_checkpoint(L, D, vocab=V, seed=13), device=DEV)
    state, g = start(model, 4)
    tokens, counts = torch.randint(0, V, (4, 3), generator=g).to(DEV), torch.tensor([1, 3, 0, 2], device=DEV)
    _, trace = model.forward_draft(tokens, state)
    captured = state.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.accept(captured, trace, counts)
    eager = model.accept(state.clone(), trace, counts)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, eager) and not torch.equal(eager[1], state[1])
    want = state[1:2].clone()
    model.forward_rows(tokens[1:2], want)
    close_states(eager[1:2], want)


def test_a_text_decoded_with_drafts_is_the_text_fed_plainly(model):
    """Draft, verify, accept, several times; then the tokens that came out are fed one after another from the first state."""
    B, K, rounds = 6, 3, 5
    state, g = start(model, B, seed=4)
    first, last = state.clone(), torch.randint(0, V, (B, 1), generator=g).to(DEV)
    texts = [[int(x)] for x in last[:, 0]]
    seen = set()
    for _ in range(rounds):
        # a draft that knows the target: its own weights, half of them shuffled away
        probe = model.forward_rows(last, state.clone())
        q1 = torch.softmax(probe + 0.5 * torch.randn(B, V, generator=g).to(DEV), -1)
        q = torch.stack([q1] + [torch.softmax(torch.randn(B, V, generator=g).to(DEV), -1)] * (K - 1), 1)
        tokens = torch.multinomial(q.reshape(B * K, V).cpu(), 1, generator=g).reshape(B, K).to(DEV)
        logits, trace = model.forward_draft(torch.cat([last, tokens], 1), state)
        _, p = ops.sample_typical(logits.reshape(B * (K + 1), V), 0.9, 0.95, u=torch.rand(B * (K + 1), device=DEV), return_probs=True)
        u = torch.rand(B, K + 1, generator=g).to(DEV)
        p = p.reshape(B, K + 1, V)
        out, accepted = ops.verify_drafts(p, q, tokens, u)
        want = rule(p.cpu().numpy(), q.cpu().numpy(), tokens.cpu().numpy(), u.cpu().numpy())
        assert np.array_equal(out.cpu().numpy(), want[0]) and np.array_equal(accepted.cpu().numpy(), want[1])
        model.accept(state, trace, accepted + 1)
        last = out.gather(1, accepted.unsqueeze(1))
        for b in range(B):
            n = int(accepted[b])
            seen.add(n)
            texts[b] += out[b, :n + 1].tolist()
    assert len(seen) > 1
    plain = first.clone()
    for b in range(B):
        want = model.forward_rows(torch.tensor([texts[b][:-1]], device=DEV), plain[b:b + 1])
        got = model.forward_rows(last[b:b + 1], state[b:b + 1].clone())
        want = model.forward_rows(torch.tensor([texts[b][-1:]], device=DEV), plain[b:b + 1].clone())
        assert float((got - want).abs().max()) < TOL
    close_states(state, plain)


def test_adapters_projection_sampler_and_verification_together():
    """Rows of several requests through a shared uint8 projection, their own adapters, the sampler's weights and the verification."""
    B, K, k, n, rank = 12, 3, 256, 1031, 8
    g = torch.Generator().manual_seed(3)
    head = quantize_fastquant(torch.randn(n, k, generator=g) * 0.1).to(DEV)
    x = torch.randn(B * (K + 1), k, generator=g).to(DEV)
    bank = ops.pack_adapters([(torch.randn(rank, k, generator=g) / 16, torch.randn(n, rank, generator=g) * 0.5, 0.5 + i) for i in range(4)],
                             torch.bfloat16, DEV)
    ids = torch.randint(-1, 4, (B,), generator=g).to(DEV)
    base = ops.gemm_u8([head], [x])[0]
    logits = ops.adapt_rows([bank], [x], ids, [base], [torch.empty_like(base)])[0]
    want = base.double().clone()
    for b, i in enumerate(ids.tolist()):
        if i >= 0:
            at = slice(b * (K + 1), (b + 1) * (K + 1))
            want[at] += float(bank[2][i]) * (x[at].double() @ bank[0][i].double().T) @ bank[1][i].double().T
    # sums of 256 and 8 products of magnitude below 20: (3 256 / 16 + 32 + 3) 2^-23 of them
    assert float((logits.double() - want).abs().max()) < 20 * 83 * 2.0 ** -23 + 2.0 ** -22 * float(want.abs().max())
    ops.adapt_rows([bank], [x], ids, [base])
    assert torch.equal(base, logits)                         # in place
    _, p = ops.sample_typical(logits, 0.8, 0.9, u=torch.rand(B * (K + 1), device=DEV), return_probs=True)
    p = p.reshape(B, K + 1, n)
    tokens = torch.multinomial(p[:, :K].reshape(B * K, n).cpu(), 1, generator=g).reshape(B, K).to(DEV)
    u = torch.rand(B, K + 1, generator=g).to(DEV)
    for q in (p[:, :K] * 2, None):
        out, accepted = ops.verify_drafts(p, q, tokens, u)
        rout, racc = rule(p.cpu().numpy(), None if q is None else q.cpu().numpy(), tokens.cpu().numpy(), u.cpu().numpy())
        assert np.array_equal(out.cpu().numpy(), rout) and np.array_equal(accepted.cpu().numpy(), racc)
        if q is not None:
            assert int(accepted.min()) == K                  # drafted from the target's own weights


def test_refusals(model):
    state, _ = start(model, 2)
    tokens = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    for bad in [(tokens[0], state), (tokens[:, :0], state), (tokens, state[:1]), (tokens, state.double()),
                (torch.zeros(2, model.rows_per_call, dtype=torch.int64, device=DEV), state)]:
        with pytest.raises(ValueError):
            model.forward_draft(*bad)
    logits, trace = model.forward_draft(tokens, state)
    with pytest.raises(ValueError):
        model.accept(state, trace, torch.ones(2, device=DEV))
    L_ = _lib.lib()
    assert L_.b200rwkv_forward_rows_draft(None, None, 1, 1, None, 0, None, None, None, 0, None) == _lib.EINVAL
    assert b"forward_rows_draft" in L_.b200rwkv_last_error()
