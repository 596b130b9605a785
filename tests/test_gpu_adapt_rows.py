"""Low-rank adapters beside shared projections (``ops.adapt_rows``) against the formula in 64 bits.

The bound of every element follows from the arithmetic: h = x A^T is a sum of K exact products (pieces of 8 bits) in fp32, in
at most 3 K / 16 + 32 additions that may each lose a unit in the last place (2^-23 of the running sum, which the sum of
magnitudes bounds); what the pieces leave out is below 2^-21 of a product; the second product the same with the rank in K's
place; y + delta is rounded once (fp32 2^-24, bf16 2^-8, fp16 2^-11 of the value; subnormal halves half of 2^-24).  For 16-bit rows h goes in with 16 of
its bits (2^-15), and with fp16 weights products of two second pieces are left out (2^-14)."""
import ctypes as C

import pytest
import torch

from rwkvstic_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(streams, T, k, outs, rank, adapters, w, t, seed=0, none=0.2):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, std=1.0: torch.randn(*s, generator=g) * std
    banks = [(rnd(adapters, rank, k, std=k ** -0.5).to(w).to(DEV), rnd(adapters, o, rank, std=rank ** -0.5).to(w).to(DEV),
              (torch.rand(adapters, generator=g) + 0.5).to(DEV)) for o in outs]
    ids = torch.randint(0, adapters, (streams,), generator=g)
    ids[torch.rand(streams, generator=g) < none] = -1
    xs = [rnd(streams * T, k).to(t).to(DEV) for _ in outs]
    ys = [rnd(streams * T, o).to(t).to(DEV) for o in outs]
    return banks, xs, ids.to(DEV), ys


def reference(bank, x, ids, y):
    """(result, bound) in fp64."""
    a, b, scale = bank
    n, T = a.shape[0], x.shape[0] // ids.shape[0]
    want, bound = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    k, rank = a.shape[2], a.shape[1]
    half = y.dtype != torch.float32
    c1 = (3 * k / 16 + 32) * 2.0 ** -23 + 2.0 ** -21
    c2 = (3 * rank / 16 + 8) * 2.0 ** -23 + (2.0 ** -15 + (2.0 ** -14 if a.dtype == torch.float16 else 0.0) if half else 2.0 ** -21)
    for i, j in enumerate(ids.tolist()):
        if not 0 <= j < n:
            continue
        at = slice(i * T, (i + 1) * T)
        s = 1.0 if scale is None else float(scale[j])
        h = x[at].double() @ a[j].double().T
        hm = x[at].double().abs() @ a[j].double().abs().T
        want[at] += s * (h @ b[j].double().T)
        bound[at] = s * ((c1 * hm + c2 * h.abs()) @ b[j].double().abs().T)
    eps = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[y.dtype]
    return want, bound * (1 + eps) + eps * want.abs() + (2.0 ** -25 if y.dtype == torch.float16 else 1e-38)


def check(banks, xs, ids, ys, outs=None, untouched=True):
    wants = [reference(b, x, ids, y) for b, x, y in zip(banks, xs, ys)]
    before = [y.clone() for y in ys]
    got = ops.adapt_rows(banks, xs, ids, ys, outs)
    torch.cuda.synchronize()
    n, T = banks[0][0].shape[0], xs[0].shape[0] // ids.shape[0]
    none = ~((ids >= 0) & (ids < n)).repeat_interleave(T)
    for y0, y, o, g, (want, bound) in zip(before, ys, outs or ys, got, wants):
        assert g is o
        assert torch.equal(g[none], y0[none])
        err = ((g.double() - want).abs() - bound)[~none]           # rows without an adapter may hold infinities; they were compared above
        assert err.numel() == 0 or float(err.max()) <= 0.0, float(err.max())
        if outs is not None and untouched:
            assert torch.equal(y, y0)


COMBOS = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")]
SHAPES = [
    (1, 1, 128, [64, 64, 128], 4, 1),        # one row, three projections
    (1, 1, 2048, [2048], 16, 3),             # K cut over CTAs
    (7, 1, 768, [770, 3], 8, 2),             # few rows of shared adapters, odd outputs
    (40, 1, 264, [130], 20, 1),              # one adapter for more rows than a tile
    (150, 1, 136, [64], 12, 40),
    (1100, 1, 64, [36], 8, 3),               # more streams than a window
    (1300, 3, 64, [36], 8, 5),               # the same with tiles that begin and end inside a stream
    (48, 5, 256, [1029], 8, 20),             # tiles that begin and end inside a stream
    (33, 31, 72, [65, 1], 4, 2),
    (3, 33, 128, [100], 36, 2),
    (1, 63, 512, [256], 64, 1),
    (2, 64, 128, [132], 100, 2),             # tiles of one stream
    (3, 65, 200, [67], 128, 3),
    (2, 333, 1024, [260, 64], 64, 5),
    (2, 70, 8, [5], 256, 2),                 # the shortest K, the largest rank
    (9, 2, 520, [1], 200, 4),
    (3, 129, 64, [1024, 392, 8], 20, 2),     # tiles of 128 rows, several matrices and columns that end inside a step
    (5, 200, 456, [640, 2048], 64, 4),
    (2, 701, 2048, [256], 128, 2),
    (40, 64, 128, [776], 48, 3),             # more tiles than SMs have steps for at once
    (1, 2000, 96, [1160, 16], 12, 1),
]


@pytest.mark.parametrize("w,t", COMBOS)
@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}_k{s[2]}_r{s[4]}" for s in SHAPES])
def test_against_formula(shape, w, t):
    banks, xs, ids, ys = make(*shape, TYPES[w], TYPES[t], seed=len(str(shape)))
    check(banks, xs, ids, ys, [torch.full_like(y, 7.0) for y in ys])
    check(banks, xs, ids, ys)


# Streams of 64 rows and more whose products are many enough for the tiles of 128 rows, in every type.
TILES = [
    (3, 1029, 1016, [1024, 392, 8], 100, 2),     # several matrices, a last tile of 5 rows, columns that end inside a step
    (40, 64, 3208, [2000], 48, 3),               # half a tile per stream, more tiles than SMs
    (1, 2000, 12008, [7520], 12, 1),
    (2, 701, 2400, [5400], 128, 2),
    (3, 129, 8200, [10000], 128, 3),             # K cut over CTAs, a tile of one row
    (6, 200, 2056, [1000, 136, 4096], 68, 4),
    (64, 300, 1304, [808], 4, 2),
    (9, 1000, 272, [64], 256, 2),                # only the first launch
    (2, 700, 8, [8192], 64, 2),                  # only the second
    (4, 500, 2048, [2049], 32, 2),               # rows that start anywhere
]


@pytest.mark.parametrize("w,t", COMBOS)
@pytest.mark.parametrize("shape", TILES, ids=[f"{s[0]}x{s[1]}_k{s[2]}_r{s[4]}" for s in TILES])
def test_tiles_against_formula(shape, w, t):
    banks, xs, ids, ys = make(*shape, TYPES[w], TYPES[t], seed=len(str(shape)))
    check(banks, xs, ids, ys, [torch.full_like(y, 7.0) for y in ys])
    check(banks, xs, ids, ys)


@pytest.mark.parametrize("w,t", COMBOS)
def test_rows_without_adapter_are_not_read(w, t):
    """Their x may hold anything, and ids outside the bank mean none."""
    banks, xs, ids, ys = make(12, 3, 64, [40], 8, 3, TYPES[w], TYPES[t], none=0.0)
    ids[2], ids[5], ids[7], ids[11] = -1, 3, -(2 ** 40), 2 ** 40
    for i in (2, 5, 7, 11):
        xs[0][3 * i:3 * i + 3] = float("nan")
        ys[0][3 * i] = float("inf")
    outs = [torch.zeros_like(ys[0])]
    check(banks, xs, ids, ys, outs)
    ids.fill_(-1)
    check(banks, xs, ids, ys, outs)
    check(banks, xs, ids, ys)


def test_no_scale_means_one_and_infinite_inputs_give_nan():
    banks, xs, ids, ys = make(3, 1, 128, [64], 8, 2, torch.bfloat16, torch.float32, none=0.0)
    banks = [(a, b, None) for a, b, _ in banks]
    check(banks, xs, ids, ys, [torch.empty_like(ys[0])])
    xs[0][1, 17] = float("inf")
    out = ops.adapt_rows(banks, xs, ids, ys, [torch.empty_like(ys[0])])[0]
    assert torch.isnan(out[1]).all() and not torch.isnan(out[[0, 2]]).any()


def test_unaligned_rows_of_y():
    """y and out may start anywhere: four elements at a time only where both allow it."""
    banks, xs, ids, ys = make(5, 2, 64, [68], 8, 2, torch.bfloat16, torch.float32)
    flat = torch.zeros(10 * 68 + 3, device=DEV)
    flat[3:] = ys[0].reshape(-1)
    y = flat[3:].reshape(10, 68)
    check(banks, xs, ids, [y], [torch.empty_like(ys[0])])
    check(banks, xs, ids, [y])
    assert float(flat[:3].abs().sum()) == 0.0


def test_extreme_values():
    """Large and small activations keep their relative accuracy (pieces share the float's exponent range)."""
    for scale in (1e30, 1e-30):
        banks, xs, ids, ys = make(4, 3, 256, [64], 16, 2, torch.bfloat16, torch.float32)
        xs = [x * scale for x in xs]
        ys = [y * scale for y in ys]
        check(banks, xs, ids, ys, [torch.empty_like(ys[0])])


def test_repeats_its_bits_and_rows_do_not_depend_on_their_tile():
    banks, xs, ids, ys = make(64, 1, 512, [300], 16, 4, torch.bfloat16, torch.float32)
    outs = [torch.empty_like(ys[0])]
    first = ops.adapt_rows(banks, xs, ids, ys, outs)[0].clone()
    for _ in range(3):
        assert torch.equal(ops.adapt_rows(banks, xs, ids, ys, outs)[0], first)
    turn = torch.randperm(64, generator=torch.Generator().manual_seed(1)).to(DEV)
    moved = ops.adapt_rows(banks, [xs[0][turn].contiguous()], ids[turn].contiguous(), [ys[0][turn].contiguous()], outs)[0]
    assert torch.equal(moved, first[turn])


def test_captured_call_follows_its_ids():
    banks, xs, ids, ys = make(6, 2, 128, [64, 33], 8, 3, torch.bfloat16, torch.bfloat16)
    outs = [torch.empty_like(y) for y in ys]
    ops.adapt_rows(banks, xs, ids, ys, outs)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            ops.adapt_rows(banks, xs, ids, ys, outs)
    for seed in range(3):
        ids.copy_(torch.randint(-1, 3, (6,), generator=torch.Generator().manual_seed(seed)))
        want = [o.clone() for o in ops.adapt_rows(banks, xs, ids, ys, [torch.empty_like(y) for y in ys])]
        for g in graphs:
            for o in outs:
                o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_two_streams_at_once():
    cases = [make(32, 1, 1024, [512], 16, 8, torch.bfloat16, torch.float32, seed=s) for s in range(2)]
    want = [ops.adapt_rows(b, x, i, y, [torch.empty_like(y[0])])[0] for b, x, i, y in cases]
    outs = [[torch.empty_like(c[3][0])] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for (b, x, i, y), o, s in zip(cases, outs, streams):
            with torch.cuda.stream(s):
                ops.adapt_rows(b, x, i, y, o)
    torch.cuda.synchronize()
    assert all(torch.equal(o[0], w) for o, w in zip(outs, want))


@pytest.mark.parametrize("shape", [(4, 1, 512, [256, 256], 16, 3), (70, 1, 512, [256, 256], 16, 3), (3, 300, 2048, [2048, 512], 64, 3)],
                         ids=["one launch", "gathered", "tiles"])
def test_every_form_captured_beside_other_calls(shape):
    """A captured call replayed on one stream while eager calls of the same shape run on another."""
    cases = [make(*shape, torch.bfloat16, torch.float32, seed=s) for s in range(2)]
    want = [[o.clone() for o in ops.adapt_rows(b, x, i, y, [torch.empty_like(v) for v in y])] for b, x, i, y in cases]
    outs = [[torch.empty_like(v) for v in c[3]] for c in cases]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adapt_rows(*cases[0], outs[0])
    other = torch.cuda.Stream()
    for _ in range(10):
        graph.replay()
        with torch.cuda.stream(other):
            ops.adapt_rows(*cases[1], outs[1])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_outputs_that_overlap_are_refused():
    banks, xs, ids, ys = make(4, 2, 64, [32, 32], 8, 2, torch.bfloat16, torch.float32)
    flat = torch.zeros(4096, device=DEV)
    near = [flat[:256].view(8, 32), flat[128:384].view(8, 32)]
    for y, out in (([ys[0], ys[0]], [ys[0], ys[0]]), (ys, [ys[1], ys[0]]), (ys, near), ([near[0], ys[1]], [near[1], ys[1]])):
        with pytest.raises(_lib.B200RWKVError, match="overlaps"):
            ops.adapt_rows(banks, xs, ids, y, out)
    square, xs, ids, ys = make(4, 2, 64, [64], 8, 2, torch.bfloat16, torch.float32)
    with pytest.raises(_lib.B200RWKVError, match="overlaps"):
        ops.adapt_rows(square, xs, ids, ys, xs)
    side = [flat[:512].view(8, 64), flat[512:1024].view(8, 64)]        # next to each other is fine
    ops.adapt_rows(square * 2, xs * 2, ids, side)


def test_pack_adapters_of_different_ranks():
    g = torch.Generator().manual_seed(5)
    parts = [(torch.randn(r, 64, generator=g) / 8, torch.randn(40, r, generator=g) / 2, 0.25 * (r + 1)) for r in (3, 8, 1)]
    bank = ops.pack_adapters(parts, torch.bfloat16, DEV)
    assert tuple(bank[0].shape) == (3, 8, 64) and tuple(bank[1].shape) == (3, 40, 8)
    x, y = torch.randn(6, 64, generator=g).to(DEV), torch.randn(6, 40, generator=g).to(DEV)
    ids = torch.tensor([2, 0, 1], device=DEV)
    check([bank], [x], ids, [y], [torch.empty_like(y)])
    for i, j in enumerate(ids.tolist()):
        a, b, s = parts[j]
        want = y[2 * i:2 * i + 2].double().cpu() + s * x[2 * i:2 * i + 2].cpu().double() @ a.bfloat16().double().T @ b.bfloat16().double().T
        got = ops.adapt_rows([bank], [x], ids, [y], [torch.empty_like(y)])[0][2 * i:2 * i + 2].double().cpu()
        assert float((got - want).abs().max()) < 1e-5       # (3 64 / 16 + 32) 2^-23 of sums of magnitude below 2


def test_refusals():
    banks, xs, ids, ys = make(4, 2, 64, [32], 8, 2, torch.bfloat16, torch.float32)
    a, b, s = banks[0]
    bad = [
        dict(banks=[]), dict(xs=[]), dict(banks=banks * 4, xs=xs * 4, ys=ys * 4),
        dict(banks=[(a.double(), b.double(), s)]), dict(xs=[xs[0].half()]), dict(ys=[ys[0].bfloat16()]),
        dict(ids=ids.int()), dict(ids=ids[:3]), dict(ids=ids.cpu()), dict(ids=ids.repeat(2)[::2]),
        dict(banks=[(a, b[:, :, :4].contiguous(), s)]), dict(banks=[(a[:1], b, s)]), dict(banks=[(a, b, s.double())]), dict(banks=[(a, b, s[:1])]),
        dict(xs=[xs[0][:, :56].contiguous()]), dict(ys=[ys[0][:, :31].contiguous()]), dict(outs=[ys[0][:4]]),
        dict(xs=[xs[0].t().contiguous().t()]), dict(banks=[(a.transpose(1, 2).contiguous().transpose(1, 2), b, s)]),
    ]
    for change in bad:
        args = {**dict(banks=banks, xs=xs, ids=ids, ys=ys, outs=None), **change}
        with pytest.raises(ValueError):
            ops.adapt_rows(args["banks"], args["xs"], args["ids"], args["ys"], args["outs"])
    with pytest.raises(RuntimeError):
        ops.adapt_rows([(a.cpu(), b.cpu(), s.cpu())], [xs[0].cpu()], ids.cpu(), [ys[0].cpu()])
    for rank, k in ((6, 64), (260, 64), (8, 60)):
        with pytest.raises(_lib.B200RWKVError):
            ops.adapt_rows([(torch.zeros(2, rank, k, device=DEV), torch.zeros(2, 32, rank, device=DEV), None)], [torch.zeros(8, k, device=DEV)],
                           ids, [torch.zeros(8, 32, device=DEV)])
    empty = torch.zeros(0, 64, device=DEV)
    assert ops.adapt_rows(banks, [empty], ids, [torch.zeros(0, 32, device=DEV)])[0].shape == (0, 32)
    assert ops.adapt_rows(banks, [empty], ids[:0], [torch.zeros(0, 32, device=DEV)])[0].shape == (0, 32)


# (streams, rows of a stream, k, outputs, rank) that take each form
FORMS = {"one launch": (3, 1, 64, 64, 8), "gathered": (70, 2, 64, 264, 16), "gathered, 32 ranks a stage": (70, 2, 64, 264, 100),
         "tiles": (2, 701, 4288, 4096, 64), "tiles, second launch of two times 64 ranks": (1, 300, 64, 8192, 128)}


@pytest.mark.parametrize("w", ["bf16", "f16"])
@pytest.mark.parametrize("form", FORMS)
def test_h_keeps_24_bits_beside_rows_of_16(form, w):
    """Pairs of 2^20 + a and -2^20 + b, which cancel in the second product: every number on the way is a whole one below 2^24
    and the result below 2^8, so it is exact.  (h in 16 bits would lose all of a and b.)"""
    streams, T, k, n_out, rank = FORMS[form]
    g = torch.Generator().manual_seed(rank)
    whole = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).double()
    a, b = torch.zeros(2, rank, k, dtype=torch.float64), torch.zeros(2, n_out, rank // 2, 2, dtype=torch.float64)
    a[:, 0::2, 0], a[:, 1::2, 0], a[:, :, k - 1] = 512.0, -512.0, whole(-7, 7, 2, rank)
    b.scatter_(2, torch.rand(2, n_out, rank // 2, generator=g).topk(4).indices.unsqueeze(-1).expand(-1, -1, -1, 2), 1.0)     # four pairs a column
    b = b.reshape(2, n_out, rank) * (2 * whole(0, 1, 2, n_out, 1) - 1)
    x, y = torch.zeros(streams * T, k, dtype=torch.float64), whole(-60, 60, streams * T, n_out)
    x[:, 0], x[:, k - 1] = 2048.0, whole(1, 3, streams * T)
    ids = torch.arange(streams) % 2
    want = y.clone()
    for i, j in enumerate(ids.tolist()):
        want[i * T:(i + 1) * T] += x[i * T:(i + 1) * T] @ a[j].T @ b[j].T
    assert float(want.abs().max()) <= 256
    d = lambda v: v.to(TYPES[w]).to(DEV)
    got = ops.adapt_rows([(d(a), d(b), None)], [d(x)], ids.to(DEV), [d(y)])[0]
    assert torch.equal(got.double().cpu(), want)


@pytest.mark.parametrize("shape", [(256, 1, 4096, [256, 256, 256], 32, 8), (40, 2, 64, [8], 4, 2), (2, 701, 4288, [64], 64, 2), (3, 700, 8, [8192], 64, 2)],
                         ids=["gathered", "small", "first launch tiles", "second launch tiles"])
def test_a_call_without_adapters_is_over_before_what_follows_it(shape):
    """No row has an adapter, so nobody needs the first launch; the call still ends with it: ids that the next operation on the stream
    fills in are not followed, and nothing is written to the workspace."""
    banks, xs, ids, ys = make(*shape, torch.bfloat16, torch.float32)
    streams, T, k, outs, rank, n = shape
    L, m = _lib.lib(), len(outs)
    bank = (_lib.Adapters * m)(*[_lib.Adapters(a.data_ptr(), b.data_ptr(), s.data_ptr(), o) for (a, b, s), o in zip(banks, outs)])
    bf16, f32 = ops._DENSE_DTYPES[torch.bfloat16], ops._DENSE_DTYPES[torch.float32]
    nbytes = L.b200rwkv_adapt_rows_workspace_bytes(m, bank, n, rank, k, bf16, streams, T)
    ws = torch.full((nbytes,), 0xA5, dtype=torch.uint8, device=DEV)
    p = lambda ts: (C.c_void_p * m)(*[t.data_ptr() for t in ts])
    px, py = p(xs), p(ys)
    before = [y.clone() for y in ys]
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(100):
        ids.fill_(-1)
        _lib.check(L.b200rwkv_adapt_rows(m, C.addressof(bank), n, rank, k, bf16, C.addressof(px), C.addressof(py), C.addressof(py), f32,
                                         ids.data_ptr(), streams, T, ws.data_ptr(), nbytes, stream))
        ids.zero_()
    torch.cuda.synchronize()
    assert all(torch.equal(y, b) for y, b in zip(ys, before))
    assert bool((ws == 0xA5).all())


def test_long_ranks_are_not_cut_off_one_after_another():
    """fp32 adapters of rank 256, all values positive, in units of 2^-23 of the whole.  A product of tensor cores cuts its terms, the running sum
    among them, to the last place of the largest, and its result: up to a unit each, half of one on average.  A chain is 32 ranks: ten
    products of small pieces, of 17 terms each, at a sum below 2^-6 of the chain's (2.7, on average 1.3), then two of the first pieces, which are
    multiples of 2^-14 below 4 and lose nothing at a sum below 128, so that running sum and result, at half and at the whole, lose 3 (1.5).
    Chains join by seven additions that round (3.5, on average 0); what is left out is below 2^-21 (4) and on average 2^-23 / 2.25 (0.5, pieces
    being spread evenly); the sum with y rounds (0.5).  One chain of 256 ranks lost 57 on average."""
    g = torch.Generator().manual_seed(3)
    rank, n_out = 256, 4096
    h, b = 1 + torch.rand(3, rank, generator=g), 1 + torch.rand(3, n_out, rank, generator=g)
    a, x = torch.zeros(3, rank, 8), torch.zeros(6, 8)
    a[:, :, 0], x[:, 0] = h, 1.0                              # h is exact: one product, of 1
    ids = torch.tensor([0, 2, 1, 0, 2, 2])
    got = ops.adapt_rows([(a.to(DEV), b.to(DEV), None)], [x.to(DEV)], ids.to(DEV), [torch.zeros(6, n_out, device=DEV)])[0].double().cpu()
    want = torch.einsum("sr,snr->sn", h[ids].double(), b[ids].double())
    lost = (want - got) / want * 2.0 ** 23
    assert float(lost.abs().max()) <= 14.0 and abs(float(lost.mean())) <= 4.0, (float(lost.abs().max()), float(lost.mean()))


def test_sizes_beyond_32_bits_are_refused():
    """They would wrap on their way to the library and be taken for small ones (2^32 + 64 for 64).  Nothing here is ever read."""
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("45 GB for the tensors")
    wide = 2 ** 32 + 64
    a, x, ids = torch.empty(1, 4, wide, dtype=torch.bfloat16, device=DEV), torch.empty(1, wide, dtype=torch.bfloat16, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    b, y = torch.zeros(1, 8, 4, dtype=torch.bfloat16, device=DEV), torch.zeros(1, 8, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="32 bits"):
        ops.adapt_rows([(a, b, None)], [x], ids, [y])
    with pytest.raises(_lib.B200RWKVError, match="k_in"):     # within 32 bits, but not in blocks of 32
        k = 2 ** 31 - 8
        ops.adapt_rows([(a.view(-1)[:4 * k].view(1, 4, k), b, None)], [x[:, :k].contiguous()], ids, [y])
    del a, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("w", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("streams,T,k,chain", [(6, 1, 4096, 32), (200, 1, 4096, 32), (3, 700, 16384, 64)], ids=["one launch", "gathered", "tiles"])
def test_long_inputs_are_not_cut_off_one_after_another(streams, T, k, chain, w):
    """The first product of rows of fp32, all values positive; units and arithmetic as above.  A chain is 32 k of a lane (tiles: 64 of a tile):
    the products of small pieces, up to five for 16 k, come first and lose 17 terms each at 2^-6 of the chain's sum; the first pieces' lose running
    sum and result only, twice for 16 k (32 k: 2 (1/2 + 1) = 3, 64 k: 2 (1/4 + 1/2 + 3/4 + 1) = 5).  Half of both on average, and 0.5 of what
    is left out (4 at most).  Chains join by additions that round, 0.5 each and 0 on average.  The second product is of h and one, exact.
    Chains of 64 and 128 k in the order of k lost 13 and 20 on average."""
    g = torch.Generator().manual_seed(5)
    a, x = (1 + torch.rand(3, 4, k, generator=g)).to(TYPES[w]), 1 + torch.rand(streams * T, k, generator=g)
    b = torch.zeros(3, 8, 4, dtype=TYPES[w])
    b[:, :, 0] = 1.0
    ids = torch.arange(streams) % 3
    got = ops.adapt_rows([(a.to(DEV), b.to(DEV), None)], [x.to(DEV)], ids.to(DEV), [torch.zeros(streams * T, 8, device=DEV)])[0].double().cpu()
    want = torch.cat([x[i * T:(i + 1) * T].double() @ a[i % 3, 0].double() for i in range(streams)]).unsqueeze(1)
    lost = (want - got) / want * 2.0 ** 23
    chains = 17 * 5 * (chain // 16) / 64 + (3 if chain == 32 else 5)
    joins = k // 256 + 16 if chain == 32 else k // 64 + 8
    assert abs(float(lost.mean())) <= chains / 2 + 0.5 and float(lost.abs().max()) <= chains + 4 + joins / 2, (float(lost.mean()), float(lost.abs().max()))
