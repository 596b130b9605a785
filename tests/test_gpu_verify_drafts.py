"""Verification of drafted tokens (``ops.verify_drafts``) against the rule written out in 64 bits, token by token."""
import numpy as np
import pytest
import torch

from rwkvstic_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rule(target, draft, tokens, u, lengths=None):
    """The definition on the host.  Weights that are not above zero count as zero."""
    target = np.where(target > 0, target, 0.0).astype(np.float64)
    draft = None if draft is None else np.where(draft > 0, draft, 0.0).astype(np.float64)
    B, K = tokens.shape
    V = target.shape[2]
    out, accepted = np.full((B, K + 1), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        n, length, w = 0, K if lengths is None else min(max(int(lengths[b]), 0), K), None
        while n < length:
            d, p, P = int(tokens[b, n]), target[b, n], target[b, n].sum()
            q = None if draft is None else draft[b, n]
            Q = 1.0 if draft is None else q.sum()
            known = 0 <= d < V
            pd, qd = p[d] if known else 0.0, (q[d] if draft is not None else 1.0) if known else 1.0
            if float(u[b, n]) * qd * P < pd * Q:
                out[b, n] = d
                n += 1
                continue
            if draft is None:
                w = p.copy()
                if known:
                    w[d] = 0.0
            else:
                w = np.maximum(p * Q - q * P, 0.0)
            if not w.sum() > 0:
                w = p
            break
        if w is None:
            w = target[b, n]
        run = np.cumsum(w)
        hit = np.nonzero((w > 0) & (run >= float(u[b, K]) * run[-1]))[0]
        some = np.nonzero(w > 0)[0]
        out[b, n] = hit[0] if hit.size else some[-1] if some.size else -1
        accepted[b] = n
    return out, accepted


def make(B, K, V, seed=0, cut=0.02):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g) * 3
    logits[:, :, 0] += 0.5 * float(np.log(V) + 4.5)
    target, draft = torch.softmax(logits, -1), torch.softmax(logits[:, :K] + 0.7 * torch.randn(B, K, V, generator=g), -1)
    target, draft = torch.where(target > cut / V, target, 0.0), torch.where(draft > cut / V, draft, 0.0)
    tokens = torch.multinomial(draft.reshape(B * K, V), 1, generator=g).reshape(B, K) if K else torch.zeros(B, 0, dtype=torch.int64)
    lengths = torch.randint(0, K + 1, (B,), generator=g)
    return target, draft, tokens, torch.rand(B, K + 1, generator=g), lengths


def check(target, draft, tokens, u, lengths=None):
    dev = lambda t: None if t is None else t.to(DEV)
    got = ops.verify_drafts(dev(target), dev(draft), dev(tokens), dev(u), dev(lengths))
    want = rule(target.numpy(), None if draft is None else draft.numpy(), tokens.numpy(), u.numpy(), None if lengths is None else lengths.numpy())
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    return want


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 50277), (3, 2, 7), (5, 3, 1023), (5, 3, 1024), (5, 3, 1025), (40, 5, 2500), (160, 2, 33), (2, 12, 20011), (20, 0, 300), (1, 64, 50),
                                   (9, 3, 9000), (80, 1, 5000)])
@pytest.mark.parametrize("drafted", [True, False])
def test_against_rule(B, K, V, drafted):
    target, draft, tokens, u, lengths = make(B, K, V, seed=B + K)
    for n in (None, lengths):
        check(target, draft if drafted else None, tokens, u, n)


def test_every_length_accepts_and_refuses():
    target, draft, tokens, u, lengths = make(300, 4, 600, seed=3)
    _, accepted = check(target, draft, tokens, u)
    assert set(accepted.tolist()) == {0, 1, 2, 3, 4}


def test_borders():
    """Numbers of 0, tokens of no weight, rows of no weight, tokens outside the vocabulary, equal distributions."""
    target, draft, tokens, u, _ = make(8, 3, 200, seed=1)
    u[0], u[1, 3], u[2] = 0.0, 0.0, 1.0 - 2.0 ** -24
    target[1, 0, tokens[1, 0]] = 0.0                          # refused whatever its number
    u[1, 0] = 0.0
    tokens[2, 1], tokens[3, 0], tokens[4, 2] = -1, 200, 2 ** 40
    target[5, 0] = 0.0                                        # nothing to draw from: -1
    draft[6, 0] = 0.0                                         # nothing drafted: the target's own
    draft[7] = 3.0 * target[7, :3]                            # the same distribution: all accepted
    tokens[7] = target[7, :3].argmax(-1)
    for d in (draft, None):
        out, accepted = check(target, d, tokens, u)
        assert out[5, 0] == -1 and accepted[5] == 0
    out, accepted = check(target, draft, tokens, u)
    assert accepted[7] == 3 and out[1, 0] != tokens[1, 0]
    one = torch.zeros(1, 2, 200)
    one[:, :, 17] = 2.0                                       # all weight on the refused token: there is nothing else to draw
    out, accepted = check(one, None, torch.tensor([[17]]), torch.tensor([[0.5, 0.5]]))
    assert accepted[0] == 1
    out, _ = check(one, one[:, :1] * 2, torch.tensor([[3]]), torch.tensor([[0.5, 0.5]]))
    assert out[0].tolist() == [17, -1]                        # token 3 has no weight; what remains is empty, so the target's own


def test_weights_that_are_not_above_zero():
    target, draft, tokens, u, _ = make(6, 2, 300, seed=9)
    target[0, 0, :50], target[1, 1, 7], draft[2, 0, 9] = -1.0, float("nan"), float("nan")
    draft[3, 1, ::2] = -0.0
    check(target, draft, tokens, u, torch.tensor([-5, 2, 1, 2, 2 ** 40, 0]))


def test_rows_behind_the_length_are_not_looked_at():
    target, draft, tokens, u, _ = make(4, 3, 100, seed=2)
    lengths = torch.tensor([0, 1, 2, 3])
    want = check(target, draft, tokens, u, lengths)
    for b, n in enumerate(lengths.tolist()):
        target[b, n + 1:], draft[b, n:], tokens[b, n:] = float("nan"), float("inf"), 2 ** 50
    got = ops.verify_drafts(target.to(DEV), draft.to(DEV), tokens.to(DEV), u.to(DEV), lengths.to(DEV))
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])


def test_strided_streams_and_rows():
    target, draft, tokens, u, lengths = make(5, 3, 257, seed=4)
    big = torch.zeros(5, 6, 300, device=DEV)
    big[:, :4, 1:258] = target.to(DEV)
    other = torch.zeros(3, 5, 257, device=DEV)
    other.copy_(draft.transpose(0, 1))
    got = ops.verify_drafts(big[:, :4, 1:258], other.transpose(0, 1), tokens.to(DEV), u.to(DEV), lengths.to(DEV))
    want = rule(target.numpy(), draft.numpy(), tokens.numpy(), u.numpy(), lengths.numpy())
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])


def test_a_stream_does_not_depend_on_the_others():
    target, draft, tokens, u, lengths = (t.to(DEV) for t in make(150, 3, 9000, seed=6))
    out, accepted = ops.verify_drafts(target, draft, tokens, u, lengths)
    for n in (1, 10, 60):
        at = slice(20, 20 + n)
        o, a = ops.verify_drafts(target[at], draft[at], tokens[at], u[at], lengths[at])
        assert torch.equal(o, out[at]) and torch.equal(a, accepted[at])


def test_tokens_come_out_as_the_targets():
    """What is emitted first is distributed as the target's first row, whatever was drafted."""
    V, n = 6, 40000
    g = torch.Generator().manual_seed(7)
    p, q = torch.tensor([0.3, 0.05, 0.25, 0.1, 0.1, 0.2]), torch.tensor([0.1, 0.4, 0.2, 0.0, 0.25, 0.05])
    target = p.repeat(n, 2, 1).to(DEV)
    draft = q.repeat(n, 1, 1).to(DEV)
    tokens = torch.multinomial(q, n, replacement=True, generator=g).reshape(n, 1).to(DEV)
    out, _ = ops.verify_drafts(target, draft, tokens, torch.rand(n, 2, generator=g).to(DEV))
    share = torch.bincount(out[:, 0].cpu(), minlength=V).double() / n
    assert float((share - p.double()).abs().max()) < 5 * 0.5 / n ** 0.5      # five standard deviations of a share


def test_captured_and_on_another_stream():
    target, draft, tokens, u, lengths = (t.to(DEV) for t in make(12, 3, 3000, seed=8))
    want = ops.verify_drafts(target, draft, tokens, u, lengths)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.verify_drafts(target, draft, tokens, u, lengths)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [ops.verify_drafts(target, draft, tokens, u, lengths) for _ in range(10)][-1]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    target, draft, tokens, u, lengths = (t.to(DEV) for t in make(4, 2, 30, seed=0))
    for args in [(target.double(), draft, tokens, u, lengths), (target[:, :2], draft, tokens, u, lengths), (target, draft[:, :1], tokens, u, lengths),
                 (target, draft.half(), tokens, u, lengths), (target, draft, tokens.int(), u, lengths), (target, draft, tokens, u[:, :2], lengths),
                 (target, draft, tokens, u.double(), lengths), (target, draft, tokens, u, lengths.int()), (target, draft, tokens, u, lengths[:2]),
                 (target.transpose(1, 2).contiguous().transpose(1, 2), draft, tokens, u, lengths), (target.cpu(), draft, tokens, u, lengths),
                 (target, draft.cpu(), tokens, u, lengths), (target, draft, tokens.repeat(1, 2)[:, ::2], u, lengths)]:
        with pytest.raises(ValueError):
            ops.verify_drafts(*args)
    with pytest.raises(_lib.B200RWKVError):
        ops.verify_drafts(torch.zeros(1, 66, 4, device=DEV), None, torch.zeros(1, 65, dtype=torch.int64, device=DEV), torch.zeros(1, 66, device=DEV))
    out, accepted = ops.verify_drafts(target[:0], draft[:0], tokens[:0], u[:0])
    assert out.shape == (0, 3) and accepted.shape == (0,)


@pytest.mark.parametrize("V", [50, 1025, 50277])
def test_nothing_is_left_where_the_draft_equals_the_target(V):
    """Weights alike bit for bit: p Q - q P is zero for every token, so a refused one is replaced by a draw from the target's own row."""
    B, K = 12, 2
    target, _, _, u, _ = make(B, K, V, seed=V, cut=0.0)
    target *= 0.25 + torch.rand(B, K + 1, 1, generator=torch.Generator().manual_seed(V))      # any sum, the draft's the same
    tokens = target[:, :K].argmax(-1)
    tokens[0::3, 0] = -1                                      # refused since they are no tokens
    tokens[1::3, 1] = V
    for b in range(2, B, 3):                                  # refused since neither gives them any weight
        target[b, 0, tokens[b, 0]] = 0.0
    out, accepted = check(target, target[:, :K].clone(), tokens, u)
    assert accepted.tolist() == [0, 1, 0] * (B // 3)


def test_sizes_beyond_32_bits_are_refused():
    """They would wrap on their way to the library (a vocabulary of 2^32 + 5 taken for 5).  Nothing here is ever read."""
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("17 GB for the weights")
    with pytest.raises(ValueError, match="32 bits"):
        ops.verify_drafts(torch.empty(1, 1, 2 ** 32 + 5, device=DEV), None, torch.zeros(1, 0, dtype=torch.int64, device=DEV), torch.zeros(1, 1, device=DEV))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("B,K,V", [(2, 3, 524288), (1, 64, 524287), (3, 1, 262145)])
@pytest.mark.parametrize("drafted", [True, False])
def test_the_largest_sizes(B, K, V, drafted):
    target, draft, tokens, u, lengths = make(B, K, V, seed=K)
    check(target, draft if drafted else None, tokens, u, lengths)
    check(target, draft if drafted else None, tokens, u)
