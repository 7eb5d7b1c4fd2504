"""The training operators (embedding gradient, gated feed-forward backward, score head + loss gradient, gradient clipping): every one against its formula in
64 bits, with bounds that follow from the formats - a rounding is off by at most half a step (bf16 2^-8, fp16 2^-11, fp32 2^-24 of the value), a sum of c
fp32 terms by at most c 2^-24 of the sum of their magnitudes (2^-23 where a matrix instruction adds: its internal order and rounding are not specified)."""
import ctypes as C
import math

import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -133, F16: 2.0 ** -24, F32: 2.0 ** -149}          # spacing of the subnormal range
U32 = 2.0 ** -24


def within(got, want, bound):
    """|got - want| <= bound elementwise (64 bits, where `want` is); NaN nowhere"""
    want = want.double()
    got = got.detach().to(want.device).double()
    bound = bound.double().to(want.device) if torch.is_tensor(bound) else torch.full_like(want, bound)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside the bound, worst by "
                           f"{float(((got - want).abs() / bound.clamp_min(1e-300)).nan_to_num(float('inf')).max()):.3g}")


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs an MI355X"
    from videoitg_amd import ops as o
    return o


def randn(*shape, dtype=F32, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype)


def strided(t, extra):
    """the same matrix on the device with `extra` columns of filler behind every row"""
    if not extra:
        return t.cuda()
    big = torch.full((t.shape[0], t.shape[1] + extra), 7.0, dtype=t.dtype, device="cuda")
    big[:, :t.shape[1]] = t.cuda()
    return big[:, :t.shape[1]]


# ---- embedding -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("table_dtype,out_dtype", [(F16, F32), (BF16, BF16), (F32, F16), (F16, F16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("n,d,vocab,extra", [(1, 4, 1, 0), (7, 12, 5, 0), (60, 3584, 320, 0), (33, 256, 64, 8), (300, 132, 700, 4), (5, 4224, 9, 0)])
def test_embed_lookup(ops, table_dtype, out_dtype, n, d, vocab, extra):
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, vocab, (n,), generator=g)
    ids[::3] = torch.tensor([-200, vocab, -1, 2 ** 40])[torch.randint(0, 4, (len(ids[::3]),), generator=g)]
    ids[-1] = vocab - 1
    table = randn(vocab, d, dtype=table_dtype, scale=0.3)
    out = strided(torch.full((n, d), 3.0, dtype=out_dtype), extra)
    got = ops.embed_lookup(ids.cuda(), strided(table, extra), out, scale=1.7)
    assert got is out
    known = (ids >= 0) & (ids < vocab)
    scale = float(torch.tensor(1.7, dtype=F32))
    want = torch.where(known[:, None], table[torch.where(known, ids, 0)].double() * scale, 0.0)
    within(out, want, want.abs() * (U32 + HALF[out_dtype]) * 1.001 + TINY[out_dtype])
    if extra:
        assert (torch.as_strided(out, (n, extra), (d + extra, 1), d) == 7.0).all()    # the columns behind the rows keep their contents
    plain = ops.embed_lookup(ids.cuda(), strided(table, extra), torch.empty(n, d, dtype=table_dtype, device="cuda"))
    assert torch.equal(plain.cpu()[known], table[ids[known]])                         # scale 1, same type: the table's own bits


def _embed_grad_want(ids, dout, vocab, scale):
    known = (ids >= 0) & (ids < vocab)
    at, rows = ids[known], dout[known].double()
    want = torch.zeros(vocab, dout.shape[1], dtype=torch.float64).index_add_(0, at, rows)
    mass = torch.zeros_like(want).index_add_(0, at, rows.abs())
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, at, torch.ones(len(at), dtype=torch.float64))
    return want * scale, mass * abs(scale), count[:, None]


IDS = {"spread": lambda n, v, g: torch.randint(0, v, (n,), generator=g),
       "one_id": lambda n, v, g: torch.full((n,), v - 1),
       "none": lambda n, v, g: torch.where(torch.arange(n) % 2 == 0, -200, v),
       "mixed": lambda n, v, g: torch.where(torch.rand(n, generator=g) < 0.5, v // 2, torch.randint(-3, v + 3, (n,), generator=g)),
       "descending": lambda n, v, g: (v - 1 - torch.arange(n) * v // n).clamp(0, v - 1)}


@pytest.mark.gpu
@pytest.mark.parametrize("ids_kind", list(IDS))
@pytest.mark.parametrize("n,d,vocab", [(1, 4, 1), (2, 12, 1), (16, 64, 511), (17, 64, 512), (333, 260, 513), (2049, 96, 320), (5003, 132, 1000)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embed_backward(ops, ids_kind, n, d, vocab, accumulate):
    g = torch.Generator().manual_seed(n + vocab)
    ids = IDS[ids_kind](n, vocab, g).long()
    dout = randn(n, d, dtype=F32, scale=0.1)
    old = randn(vocab, d, scale=0.5, seed=3)
    table = old.cuda().clone()
    ops.embed_backward(ids.cuda(), dout.cuda(), table, scale=0.5, accumulate=accumulate)
    want, mass, count = _embed_grad_want(ids, dout, vocab, 0.5)
    if accumulate:
        untouched = count[:, 0] == 0
        assert torch.equal(table.cpu()[untouched], old[untouched])
        want = want + old.double()
    within(table, want, (count + 3) * U32 * mass + U32 * want.abs() * 2)
    again = old.cuda().clone()
    ops.embed_backward(ids.cuda(), dout.cuda(), again, scale=0.5, accumulate=accumulate)
    assert torch.equal(again, table)                                                   # a fixed summation order


@pytest.mark.gpu
@pytest.mark.parametrize("dout_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("table_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embed_backward_types_and_strides(ops, dout_dtype, table_dtype, accumulate):
    n, d, vocab = 700, 136, 90
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(-2, vocab - 7, (n,), generator=g)
    dout, old = randn(n, d, dtype=dout_dtype, scale=0.1), randn(vocab, d, dtype=table_dtype, scale=0.5)
    for extra in (0, 4, 8):
        table = strided(old, extra)
        ops.embed_backward(ids.cuda(), strided(dout, extra), table, scale=2.0, accumulate=accumulate)
        want, mass, count = _embed_grad_want(ids, dout, vocab, 2.0)
        if accumulate:
            want = want + old.double()
        within(table, want, (count + 4) * U32 * (mass + want.abs()) + HALF[table_dtype] * want.abs() * 1.001 + TINY[table_dtype])
        if extra:                                                                      # the columns behind the rows keep their contents
            behind = torch.as_strided(table, (vocab, extra), (d + extra, 1), d)
            assert (behind == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab,kind", [(15360, 9000, "mixed"), (15361, 9000, "mixed"), (15361, 400, "none"), (70001, 300000, "mixed"), (40000, 3, "spread"), (33000, 152064, "one_id"), (65536, 2 ** 27 - 3, "spread")])
def test_embed_backward_long_lists(ops, n, vocab, kind):
    """several digits per key, many sort tiles, runs over hundreds of chunks; the touched rows of a large vocabulary only"""
    d = 8
    g = torch.Generator().manual_seed(n)
    ids = IDS[kind](n, vocab, g).long()
    dout = randn(n, d, scale=0.1)
    known = (ids >= 0) & (ids < vocab)
    token, which = torch.unique(ids[known], return_inverse=True)
    want = torch.zeros(len(token), d, dtype=torch.float64).index_add_(0, which, dout[known].double())
    mass = torch.zeros(len(token), d, dtype=torch.float64).index_add_(0, which, dout[known].double().abs())
    table = torch.zeros(vocab, d, device="cuda")
    ops.embed_backward(ids.cuda(), dout.cuda(), table, accumulate=True)
    assert int((table != 0).any(1).sum()) == len(token)
    dense = torch.full((vocab, d), 5.0, dtype=F32, device="cuda") if vocab < 10 ** 6 else None
    if dense is not None:
        assert torch.equal(ops.embed_backward(ids.cuda(), dout.cuda(), dense), table)
    # a row's terms are added in chunks of 16, 32 or 64 and then chunk by chunk, in eight parts: far fewer roundings than n; the bound counts 32 + n / 256 + 8
    # (chunks of 64 from 32 768 tokens on: 64 + n / 512 + 8 is less)
    within(table[token.cuda()], want, (48 + n / 256) * U32 * mass)


@pytest.mark.gpu
def test_embeddings_of_millions_of_tokens(ops):
    """more rows than the lookup has blocks; a sort of thousands of tiles.  Whole numbers: every sum is exact in any order"""
    n, d, vocab = 4_300_000, 4, 300_000
    ids = torch.randint(-1, vocab, (n,), generator=torch.Generator().manual_seed(5)).cuda()
    table = torch.randint(-8, 9, (vocab, d), generator=torch.Generator().manual_seed(6)).to(F16).cuda()
    want = torch.where(ids[:, None] >= 0, table[ids.clamp(min=0)], torch.zeros((), dtype=F16, device="cuda"))
    assert torch.equal(ops.embed_lookup(ids, table, torch.full((n, d), 7.0, dtype=F16, device="cuda")), want)
    grad = torch.zeros(vocab + 1, d, dtype=torch.float64, device="cuda").index_add_(0, torch.where(ids >= 0, ids, vocab), want.double() + 1)[:vocab]
    got = ops.embed_backward(ids, want.float() + 1, torch.empty(vocab, d, device="cuda"))
    assert torch.equal(got.double(), grad)


@pytest.mark.gpu
def test_embed_backward_of_no_tokens(ops):
    table = torch.full((10, 8), 2.0, device="cuda")
    none, rows = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, 8, device="cuda")
    ops.embed_backward(none, rows, table, accumulate=True)
    assert (table == 2.0).all()
    ops.embed_backward(none, rows, table)
    assert (table == 0.0).all()
    assert ops.embed_lookup(none, table, rows).shape == (0, 8)


# ---- gated feed-forward ------------------------------------------------------------------------------------------------------------------
def halves(t):
    b = t.unflatten(-1, (-1, 2, 32))
    return b[..., 0, :].flatten(-2), b[..., 1, :].flatten(-2)


def interleave(gate, up):
    return torch.stack([gate.unflatten(-1, (-1, 32)), up.unflatten(-1, (-1, 32))], -2).flatten(-3)


FFN_SHAPES = [(1, 64, 64), (2, 128, 192), (16, 192, 320), (17, 256, 1216), (64, 64, 128), (65, 320, 64), (100, 64, 256), (255, 128, 640), (257, 192, 512),
              (400, 256, 832), (1000, 128, 1984)]


# shapes that reach the other kernels (256 CUs: at most one 128x128 tile each is the ring kernel's case): 128x128 tiles at two per CU, 256-, 320- and 384-row tiles
FFN_WIDE = [(100, 64, 33024), (200, 64, 16576), (300, 64, 12800), (300, 64, 25600), (400, 128, 12864), (1000, 64, 16384), (770, 192, 24640)]


def place(*tensors):
    """the reference's operands, 64 bits, on the device (the host would take minutes over the wide shapes)"""
    return [t.cuda().double() for t in tensors]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", FFN_SHAPES + FFN_WIDE)
@pytest.mark.parametrize("extra", [0, 8])
def test_swiglu(ops, dtype, m, k, n, extra):
    x, w = randn(m, k, dtype=dtype), randn(n, k, dtype=dtype, scale=k ** -0.5 * 1.5)
    out, gu = strided(torch.zeros(m, n // 2, dtype=dtype), extra), strided(torch.zeros(m, n, dtype=dtype), extra)
    ops.swiglu(strided(x, extra), strided(w, extra), out, gu=gu)
    x64, w64 = place(x, w)
    pre = x64 @ w64.t()
    err = k * 2.0 ** -23 * (x64.abs() @ w64.abs().t())                                 # the fp32 sums
    within(gu, pre, err + HALF[dtype] * (pre.abs() + err) * 1.001 + TINY[dtype])
    (gate, up), (eg, eu) = halves(pre), halves(err)
    silu = gate * torch.sigmoid(gate)
    # |silu'| <= 1.1; the device's exponential and reciprocal: a few units of 2^-23 each, taken as 2^-19 together
    bound = 1.1 * eg * (up.abs() + eu) + (silu.abs()) * eu + 2.0 ** -19 * (silu * up).abs()
    bound = bound + HALF[dtype] * ((silu * up).abs() + bound) * 1.001 + TINY[dtype]
    within(out, silu * up, bound)
    alone = strided(torch.zeros(m, n // 2, dtype=dtype), extra)
    ops.swiglu(strided(x, extra), strided(w, extra), alone)
    within(alone, silu * up, bound)
    if extra:
        for t, cols in ((out, n // 2), (gu, n), (alone, n // 2)):
            assert (torch.as_strided(t, (m, extra), (cols + extra, 1), cols) == 7.0).all()


def ffn_grads(dout, gu, x, w):
    """gradients in 64 bits from the saved pre-activations, and the sums of magnitudes behind them"""
    gate, up = halves(gu)
    sig = torch.sigmoid(gate)
    dgu = interleave(dout * up * sig * (1 + gate * (1 - sig)), dout * gate * sig)
    return dgu, dgu @ w, dgu.t() @ x, dgu.abs() @ w.abs(), dgu.abs().t() @ x.abs()


def check_swiglu_backward(ops, dtype, m, k, n, dw_kind, extra):
    x, w = randn(m, k, dtype=dtype), randn(n, k, dtype=dtype, scale=k ** -0.5)
    gu, dout = randn(m, n, dtype=dtype, scale=1.3, seed=1), randn(m, n // 2, dtype=dtype, scale=0.3, seed=2)
    dw_dtype = F32 if dw_kind.startswith("fp32") else dtype
    old = randn(n, k, dtype=dw_dtype, scale=0.7, seed=4)
    add = dw_kind.endswith("add")
    dx, dw = strided(torch.zeros(m, k, dtype=dtype), extra), strided(old, extra)
    ops.swiglu_backward(strided(dout, extra), strided(gu, extra), strided(x, extra), strided(w, extra), dx=dx, dw=dw, accumulate=add)
    dout64, gu64, x64, w64, old64 = place(dout, gu, x, w, old)
    dgu, want_x, want_w, mass_x, mass_w = ffn_grads(dout64, gu64, x64, w64)
    # dGU in 32 bits (2^-18 of the value: exponential, reciprocal, five products and 1 + G (1 - sig), whose cancellation is at most 4.6 in magnitude of its
    # terms over its value where dG matters; taken on the magnitude of dH U sig (1 + |G|)), then one rounding to the operand type, then the fp32 sums
    gate, up = halves(gu64)
    sig = torch.sigmoid(gate)
    fuzz = interleave((dout64 * up).abs() * sig * (1 + gate.abs()), (dout64 * gate).abs() * sig) * 2.0 ** -18 + TINY[dtype]
    ex = (HALF[dtype] * 1.01 + n * 2.0 ** -23) * mass_x + fuzz @ w64.abs()
    ew = (HALF[dtype] * 1.01 + m * 2.0 ** -23) * mass_w + fuzz.t() @ x64.abs()
    if add:
        want_w = want_w + old64
        ew = ew + m * 2.0 ** -23 * old64.abs()
    within(dx, want_x, ex + HALF[dtype] * (want_x.abs() + ex) + TINY[dtype])
    within(dw, want_w, ew + HALF[dw_dtype] * (want_w.abs() + ew) + TINY[dw_dtype])
    # independent roundings average: over the whole matrix the error is far below the worst case
    assert (dx.double() - want_x).norm() <= 2 * HALF[dtype] * want_x.norm()
    assert (dw.double() - want_w).norm() <= 2 * HALF[dtype] * want_w.norm()
    if extra:
        assert (torch.as_strided(dx, (m, extra), (k + extra, 1), k) == 7.0).all() and (torch.as_strided(dw, (n, extra), (k + extra, 1), k) == 7.0).all()
    # each alone, where another split or kernel may take it
    only_x, only_w = torch.empty(m, k, dtype=dtype, device="cuda"), old.cuda().clone()
    ops.swiglu_backward(dout.cuda(), gu.cuda(), x.cuda(), w.cuda(), dx=only_x)
    ops.swiglu_backward(dout.cuda(), gu.cuda(), x.cuda(), w.cuda(), dw=only_w, accumulate=add)
    within(only_x, want_x, ex + HALF[dtype] * (want_x.abs() + ex) + TINY[dtype])
    within(only_w, want_w, ew + HALF[dw_dtype] * (want_w.abs() + ew) + TINY[dw_dtype])
    again = torch.empty(m, k, dtype=dtype, device="cuda")
    ops.swiglu_backward(dout.cuda(), gu.cuda(), x.cuda(), w.cuda(), dx=again)
    assert torch.equal(again, only_x)                                                  # a fixed summation order


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", FFN_SHAPES + [(129, 1024, 4096), (300, 256, 8192), (33, 576, 1024), (2100, 64, 128), (3000, 320, 192), (5000, 512, 64)])
@pytest.mark.parametrize("dw_kind", ["same", "same_add", "fp32", "fp32_add"])
def test_swiglu_backward(ops, dtype, m, k, n, dw_kind):
    check_swiglu_backward(ops, dtype, m, k, n, dw_kind, 8 if m % 2 else 0)


# wider layers (256 CUs): W as it lies on 256- and 320-row tiles, whole and split; W transposed, whole (256- and 384-row tiles) and split (256, 320); dW whole
# and split on 256x256 tiles; the ring kernel on one of the two products only
@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(2100, 2048, 128), (2100, 2048, 1024), (300, 3584, 8192), (700, 4096, 6144), (4100, 2048, 2560), (3463, 320, 41344), (3177, 320, 51648),
                                   (7000, 1088, 2048), (734, 192, 16896), (900, 2048, 4096), (100, 2048, 16576), (20, 1088, 20544)])
@pytest.mark.parametrize("dtype,dw_kind", [(BF16, "same"), (F16, "fp32_add"), (BF16, "same_add")])
def test_swiglu_backward_wide(ops, dtype, m, k, n, dw_kind):
    check_swiglu_backward(ops, dtype, m, k, n, dw_kind, 8 if m % 3 == 0 else 0)


@pytest.mark.gpu
def test_swiglu_of_no_rows(ops):
    x, gu, dout = (torch.empty(0, c, dtype=F16, device="cuda") for c in (64, 128, 64))
    w = randn(128, 64, dtype=F16).cuda()
    ops.swiglu(x, w, dout, gu=gu)
    for dtype in (F16, F32):
        dw = torch.full((128, 64), 2.0, dtype=dtype, device="cuda")
        ops.swiglu_backward(dout, gu, x, w, dx=torch.empty_like(x), dw=dw, accumulate=True)
        assert (dw == 2.0).all()
        ops.swiglu_backward(dout, gu, x, w, dx=torch.empty_like(x), dw=dw)
        assert (dw == 0.0).all()


# ---- clipping --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(1,)], [(3,), (0,), (129, 7)], [(32768,), (32769,), (16384,), (65537,)], [(257, 33)] * 7, [(5,)] * 200 + [(70000,)]],
                         ids=["one", "small", "piece_edges", "seven", "many"])
@pytest.mark.parametrize("max_norm", [0.25, 1e6])
@pytest.mark.parametrize("in_place", [False, True])
def test_clip_grad_norm(ops, shapes, max_norm, in_place):
    dtypes = [F32, BF16, F16]
    grads = [randn(*s, dtype=dtypes[i % 3], scale=0.05, seed=i) for i, s in enumerate(shapes)]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in grads)) * 0.5
    dev = [t.cuda() for t in grads]
    outs = None if in_place else [torch.full_like(t, 9.0) for t in dev]
    got = ops.clip_grad_norm(dev, max_norm, outs=outs, scale=0.5)
    assert abs(got.item() - norm) <= 4 * U32 * norm
    factor = 0.5 * min(1.0, max_norm / (norm + 1e-6))
    for t, o in zip(grads, dev if in_place else outs):
        want = t.double() * factor
        within(o, want, want.abs() * (4 * U32 + HALF[t.dtype] * 1.001) + TINY[t.dtype])
    if not in_place:
        assert all(torch.equal(t.cpu(), u) for t, u in zip(dev, grads))
    alone = ops.clip_grad_norm([t.cuda() for t in grads], None, scale=0.5)
    assert torch.equal(alone, got)


@pytest.mark.gpu
def test_clip_grad_norm_of_unaligned_views(ops):
    base = {d: randn(5000, dtype=d, scale=0.1).cuda() for d in (F32, BF16, F16)}
    grads = [base[F32][1:4002], base[BF16][3:4000], base[F16][1:2], base[F16][7:4999]]
    keep = {d: t.clone() for d, t in base.items()}
    host = [t.double().cpu() for t in grads]
    norm = math.sqrt(sum(float(t.square().sum()) for t in host))
    got = ops.clip_grad_norm(grads, 0.1)
    assert abs(got.item() - norm) <= 4 * U32 * norm
    factor = 0.1 / (norm + 1e-6)
    for t, h in zip(grads, host):
        within(t, h * factor, (h * factor).abs() * (4 * U32 + HALF[t.dtype] * 1.001) + TINY[t.dtype])
    assert torch.equal(base[F32][:1], keep[F32][:1]) and torch.equal(base[F32][4002:], keep[F32][4002:])
    assert torch.equal(base[BF16][:3], keep[BF16][:3]) and torch.equal(base[F16][2:7], keep[F16][2:7])


@pytest.mark.gpu
def test_clip_grad_norm_extremes(ops):
    big = [torch.full((1000,), 3e30, device="cuda"), torch.full((10,), 1e30, dtype=BF16, device="cuda")]      # squares beyond fp32
    want = math.sqrt(1000 * float(torch.tensor(3e30).double()) ** 2 + 10 * float(torch.tensor(1e30, dtype=BF16).double()) ** 2)
    assert abs(ops.clip_grad_norm(big, 1.0).item() / want - 1) < 4 * U32
    assert abs(big[0][0].item() / (3e30 / want) - 1) < 8 * U32
    small = [torch.full((1000,), 1e-30, device="cuda")]                                                        # squares below fp32
    assert abs(ops.clip_grad_norm(small, None).item() / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    inf = [torch.tensor([1.0, float("inf")], device="cuda"), torch.ones(3, device="cuda")]
    assert ops.clip_grad_norm(inf, 1.0).item() == float("inf")
    assert inf[0][0].item() == 0.0 and math.isnan(inf[0][1].item()) and (inf[1] == 0).all()
    nan = [torch.tensor([float("nan")], device="cuda"), torch.ones(3, device="cuda")]
    assert math.isnan(ops.clip_grad_norm(nan, 1.0).item()) and nan[1].isnan().all()
    zero = [torch.zeros(5, device="cuda"), torch.empty(0, device="cuda")]
    assert ops.clip_grad_norm(zero, 1.0).item() == 0.0 and (zero[0] == 0).all()
    assert ops.clip_grad_norm([torch.empty(0, device="cuda")], 1.0).item() == 0.0
    free = [torch.full((4,), 2.0, device="cuda")]
    assert ops.clip_grad_norm(free, float("inf"), scale=0.25).item() == 1.0 and (free[0] == 0.5).all()


# ---- score head and loss ---------------------------------------------------------------------------------------------------------------
def loss_parts(z, y, scale=1.0):
    z, y, n = z.double(), y.double(), z.numel()
    pos = float(y.sum())
    pw = min(5.0, math.sqrt((n - pos) / max(1.0, pos)))
    loss = -(pw * y * torch.nn.functional.logsigmoid(z) + (1 - y) * torch.nn.functional.logsigmoid(-z)).mean()
    return loss, pw, scale / n * (torch.sigmoid(z) * (1 - y) - pw * y * torch.sigmoid(-z))


@pytest.mark.gpu
@pytest.mark.parametrize("n,p,spread", [(1, 1.0, 3.0), (1, 0.0, 3.0), (64, 0.5, 1.0), (512, 0.06, 3.0), (300, 0.004, 60.0), (2500, 0.2, 8.0), (200, 1.0, 2.0)])
def test_bce_loss_backward(ops, n, p, spread):
    g = torch.Generator().manual_seed(n)
    z, y = torch.randn(n, generator=g) * spread, (torch.rand(n, generator=g) < p).float()
    loss, pw, dz = ops.bce_loss_backward(z.cuda(), y.cuda(), scale=0.5)
    want, want_pw, want_dz = loss_parts(z, y, 0.5)
    assert abs(loss.item() - want.item()) <= 2.0 ** -20 * max(1.0, abs(want.item())) and abs(pw.item() - want_pw) <= 4 * U32 * 5
    # exponential, division, weight: a few units of 2^-24 each, 2^-20 together; fp32 has no values below 2^-149
    within(dz, want_dz, want_dz.abs() * 2.0 ** -20 + 2.0 ** -140)
    eps = 1e-4                                                                          # and against differences of the 64-bit loss
    for i in range(0, n, max(1, n // 5)):
        hi, lo = z.double().clone(), z.double().clone()
        hi[i] += eps
        lo[i] -= eps
        slope = (loss_parts(hi, y)[0] - loss_parts(lo, y)[0]).item() / (2 * eps) * 0.5
        assert abs(dz[i].item() - slope) <= 1e-6
    plain, plain_pw = ops.bce_loss(z.cuda(), y.cuda())
    assert abs(plain.item() - loss.item()) <= 1e-5 * max(1.0, abs(want.item())) and abs(plain_pw.item() - pw.item()) <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("h_dtype,dh_dtype", [(F32, F32), (BF16, BF16), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("frames,tokens,d,extra", [(1, 1, 4, 0), (3, 5, 132, 4), (17, 25, 3584, 0), (70, 1, 256, 8), (9, 81, 520, 0), (2, 3, 8200, 0), (5, 131, 520, 0), (2, 128, 3584, 4)])
def test_pool_score_and_gradients(ops, h_dtype, dh_dtype, frames, tokens, d, extra):
    h, w, b = randn(frames * tokens, d, dtype=h_dtype), randn(d, scale=d ** -0.5 * 3), randn(1)
    logits, pooled = torch.empty(frames, device="cuda"), strided(torch.zeros(frames, d), extra)
    ops.pool_score_save(strided(h, extra), frames, tokens, d, w.cuda(), b.cuda(), logits, pooled)
    mean = h.double().view(frames, tokens, d).mean(1)
    mass = h.double().abs().view(frames, tokens, d).mean(1)
    within(pooled, mean, (tokens + 3) * U32 * mass)
    within(logits, mean @ w.double() + b.double(), (tokens + d / 64 + 24) * U32 * (mass @ w.double().abs()) + 2 * U32 * b.double().abs() + 2 * U32 * (mean @ w.double()).abs())
    if h_dtype == F32 and not extra:
        plain = ops.pool_score(h.cuda(), frames, tokens, d, w.cuda(), b.cuda(), torch.empty(frames, device="cuda"))
        within(plain, logits.double().cpu(), (tokens + d) * 2.0 ** -23 * (mass @ w.double().abs()) + 2.0 ** -22)
    dz = randn(frames, scale=0.01, seed=9)
    dh = strided(torch.zeros(frames * tokens, d, dtype=dh_dtype), extra)
    old_w, old_b = randn(d, seed=11), randn(1, seed=12)
    for add in (False, True):
        dw, db = old_w.cuda().clone(), old_b.cuda().clone()
        ops.pool_score_backward(pooled, frames, tokens, d, w.cuda(), dz.cuda(), dh, dw=dw, db=db, accumulate=add)
        want = (dz.double() / tokens)[:, None, None] * w.double()
        want = want.expand(frames, tokens, d).reshape(-1, d)
        within(dh, want, want.abs() * (3 * U32 + HALF[dh_dtype] * 1.001) + TINY[dh_dtype] + 2.0 ** -149)
        terms = dz.double()[:, None] * pooled.double().cpu()
        base_w, base_b = (old_w.double(), old_b.double()) if add else (0.0, 0.0)
        want_w = terms.sum(0) + base_w
        within(dw, want_w, (frames / 16 + 19) * U32 * terms.abs().sum(0) + 2 * U32 * want_w.abs())
        want_b = dz.double().sum().reshape(1) + base_b
        within(db, want_b, 2 * U32 * (want_b.abs() + dz.double().sum().abs()))
    only = torch.empty_like(dh)
    ops.pool_score_backward(pooled, frames, tokens, d, w.cuda(), dz.cuda(), only)
    assert torch.equal(only, dh)
    db2 = torch.zeros(1, device="cuda")
    ops.pool_score_backward(pooled, frames, tokens, d, w.cuda(), dz.cuda(), db=db2)
    within(db2, dz.double().sum().reshape(1), 2 * U32 * dz.double().sum().abs())
    if extra:
        assert (torch.as_strided(dh, (frames * tokens, extra), (d + extra, 1), d) == 7.0).all()


# ---- the operators together --------------------------------------------------------------------------------------------------------------
class Step:
    """a toy selector: tokens -> embedding -> gated feed-forward -> per-frame score -> loss, and one training step's gradients, clipped"""

    def __init__(self, dtype=BF16, frames=24, tokens=5, k=128, f=64, vocab=50, seed=0):
        self.frames, self.tokens, self.k, self.f, self.vocab, self.dtype = frames, tokens, k, f, vocab, dtype
        g = torch.Generator().manual_seed(seed)
        self.ids = torch.randint(0, vocab, (frames * tokens,), generator=g)
        self.ids[::11] = -200
        self.table, self.wgu = randn(vocab, k, dtype=dtype, seed=seed), randn(2 * f, k, dtype=dtype, scale=k ** -0.5 * 2, seed=seed + 1)
        self.w, self.b = randn(f, scale=0.5, seed=seed + 2), randn(1, seed=seed + 3)
        self.labels = (torch.rand(frames, generator=g) < 0.3).float()
        rows = frames * tokens
        new = lambda *s, dt=F32: torch.empty(*s, dtype=dt, device="cuda")      # noqa: E731
        self.dev = {n: getattr(self, n).cuda() for n in ("ids", "table", "wgu", "w", "b", "labels")}
        self.x, self.h, self.gu = new(rows, k, dt=dtype), new(rows, f, dt=dtype), new(rows, 2 * f, dt=dtype)
        self.logits, self.pooled, self.dh, self.dx = new(frames), new(frames, f), new(rows, f, dt=dtype), new(rows, k, dt=dtype)
        self.dw, self.db, self.dgu, self.dtable = new(f), new(1), new(2 * f, k), new(vocab, k)

    def run(self, K):
        d = self.dev
        K.embed_lookup(d["ids"], d["table"], self.x, scale=1.5)
        K.swiglu(self.x, d["wgu"], self.h, gu=self.gu)
        K.pool_score_save(self.h, self.frames, self.tokens, self.f, d["w"], d["b"], self.logits, self.pooled)
        loss, _, dz = K.bce_loss_backward(self.logits, d["labels"], scale=64.0)
        K.pool_score_backward(self.pooled, self.frames, self.tokens, self.f, d["w"], dz, self.dh, dw=self.dw, db=self.db)
        K.swiglu_backward(self.dh, self.gu, self.x, d["wgu"], dx=self.dx, dw=self.dgu)
        K.embed_backward(d["ids"], self.dx, self.dtable, scale=1.5)
        norm = K.clip_grad_norm([self.dtable, self.dgu, self.dw, self.db], 0.05, scale=1.0 / 64.0)
        return {"loss": loss, "norm": norm, "dtable": self.dtable, "dgu": self.dgu, "dw": self.dw, "db": self.db}

    def loss64(self, table, wgu, w, b):
        known = self.ids >= 0
        x = torch.where(known[:, None], table[torch.where(known, self.ids, 0)] * 1.5, 0.0)
        gate, up = halves(x @ wgu.t())
        h = gate * torch.sigmoid(gate) * up
        return loss_parts64(h.view(self.frames, self.tokens, self.f).mean(1) @ w + b, self.labels)


def loss_parts64(z, y):
    y, n = y.double(), z.numel()
    pos = float(y.sum())
    pw = min(5.0, math.sqrt((n - pos) / max(1.0, pos)))
    return -(pw * y * torch.nn.functional.logsigmoid(z) + (1 - y) * torch.nn.functional.logsigmoid(-z)).mean()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_training_step(ops, dtype):
    from videoitg_amd.torch_ops import K
    step = Step(dtype)
    got = {n: t.clone() for n, t in step.run(K).items()}
    leaves = [t.double().requires_grad_() for t in (step.table, step.wgu, step.w, step.b)]
    loss = step.loss64(*leaves)
    grads = torch.autograd.grad(loss, leaves)
    norm = math.sqrt(sum(float(t.square().sum()) for t in grads))
    # every stored 16-bit tensor of the chain (x, gu, h, dh, dgu, dx) is off by at most half a step: six roundings and their propagation through factors of
    # order one bound the relative error of a gradient's norm by 16 half steps
    rel = 16 * HALF[dtype]
    assert abs(got["loss"].item() - loss.item()) <= rel * abs(loss.item())
    assert abs(got["norm"].item() - norm) <= rel * norm
    factor = min(1.0, 0.05 / (norm + 1e-6))
    assert factor < 1.0
    for name, want in zip(("dtable", "dgu", "dw", "db"), grads):
        err = (got[name].double().cpu().view_as(want) - want * factor).norm() / (want * factor).norm()
        assert err <= 2 * rel, (name, float(err))
    # the clipped gradient against a difference of the 64-bit loss along a random direction
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in leaves]
    eps = 1e-5
    with torch.no_grad():
        ends = [step.loss64(*[t + s * eps * d for t, d in zip(leaves, dirs)]).item() for s in (1, -1)]
    slope = (ends[0] - ends[1]) / (2 * eps) * factor
    along = sum(float((got[n].double().cpu().view_as(d) * d).sum()) for n, d in zip(("dtable", "dgu", "dw", "db"), dirs))
    size = factor * norm * math.sqrt(sum(float(d.square().sum()) for d in dirs))
    assert abs(along - slope) <= rel * size


@pytest.mark.gpu
def test_training_step_in_a_graph_and_on_another_stream(ops):
    """captured once, replayed with eager work of other data in between: every replay equals the eager result"""
    from videoitg_amd.torch_ops import K
    step, other = Step(F16, seed=5), Step(F16, seed=6)
    eager = {n: t.clone() for n, t in step.run(K).items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = {n: t.clone() for n, t in step.run(K).items()}
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for n in eager:
        assert torch.equal(eager[n], again[n]), n
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step.run(K)
    for _ in range(4):
        other.run(K)
        for t in (step.x, step.gu, step.dx, step.dtable, step.dgu, step.dw):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n in eager:
            assert torch.equal(out[n], eager[n]), n


@pytest.mark.gpu
def test_given_workspaces_of_exactly_the_planned_size(ops):
    for m, k, n in ((5, 128, 256), (300, 256, 832), (2100, 2048, 128)):
        x, w, gu, dout = (randn(*s, dtype=F16, seed=i).cuda() for i, s in enumerate(((m, k), (n, k), (m, n), (m, n // 2))))
        need = ops.swiglu_backward_plan(m, n, k)
        guard = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
        got, want = [torch.empty_like(x), torch.empty_like(w)], [torch.empty_like(x), torch.empty_like(w)]
        ops.swiglu_backward(dout, gu, x, w, dx=got[0], dw=got[1], workspace=guard[:need])
        ops.swiglu_backward(dout, gu, x, w, dx=want[0], dw=want[1])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (guard[need:] == 0x5a).all()
    for t, d in ((37, 36), (20000, 24)):
        ids, rows = torch.randint(0, 50, (t,), device="cuda"), randn(t, d).cuda()
        need = ops.embed_backward_plan(t, d)
        guard = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
        got = ops.embed_backward(ids, rows, torch.empty(50, d, device="cuda"), workspace=guard[:need])
        assert torch.equal(got, ops.embed_backward(ids, rows, torch.empty(50, d, device="cuda"))) and (guard[need:] == 0x5a).all()
    grads = [randn(70000, seed=i).cuda() for i in range(100)]
    guard = torch.full((2 * 1024 * 8 + 4096,), 0x5a, dtype=torch.uint8, device="cuda")      # two launches' sums: 96 + 4 tensors of 5 pieces
    need = (96 * 5 + 4 * 5) * 8
    norm = torch.zeros(1, device="cuda")
    assert ops.clip_grad_norm(grads, None, norm=norm, workspace=guard[:need]) is norm
    assert torch.equal(norm, ops.clip_grad_norm(grads, None)) and (guard[need:] == 0x5a).all()


@pytest.mark.gpu
def test_nan_and_infinity_stay_where_they_belong(ops):
    nan = float("nan")
    for n in (40, 20000):                                # rank sort, radix passes
        ids = torch.randint(0, 50, (n,), generator=torch.Generator().manual_seed(n)).cuda()
        ids[::3] = -200
        ids[1::7] = 50
        out = ids < 0
        out |= ids >= 50
        dout = torch.ones(n, 8, device="cuda")
        dout[out] = nan
        got = ops.embed_backward(ids, dout, torch.empty(50, 8, device="cuda"))
        assert torch.equal(got[:, 0].cpu(), torch.bincount(ids[~out], minlength=50).float().cpu())
        table = torch.full((50, 8), nan, device="cuda")
        table[:49] = 2.0
        rows = ops.embed_lookup(ids, table, torch.empty(n, 8, device="cuda"))
        assert (rows[out] == 0).all() and torch.equal(rows.isnan().any(1), ids == 49)
    for m, n, k in ((9, 128, 64), (100, 256, 192), (300, 32768, 64), (600, 1024, 128)):
        x, w, dout = randn(m, k, dtype=BF16).cuda(), randn(n, k, dtype=BF16, seed=1).cuda(), randn(m, n // 2, dtype=BF16, seed=2).cuda()
        x[m // 2], x[m - 1] = nan, float("inf")
        bad = torch.zeros(m, dtype=torch.bool, device="cuda")
        bad[m // 2] = bad[m - 1] = True
        act, gu, dx = torch.empty(m, n // 2, dtype=BF16, device="cuda"), torch.empty(m, n, dtype=BF16, device="cuda"), torch.empty_like(x)
        ops.swiglu(x, w, act, gu=gu)
        assert act[~bad].isfinite().all() and gu[~bad].isfinite().all() and not act[m // 2].isfinite().any()
        ops.swiglu_backward(dout, gu, x, w, dx=dx)
        assert dx[~bad].isfinite().all() and not dx[m // 2].isfinite().any()
    for frames, tokens in ((5, 7), (5, 200)):
        h = torch.ones(frames * tokens, 1024, device="cuda")
        h[2 * tokens + tokens // 2] = nan
        z, pooled = torch.empty(frames, device="cuda"), torch.empty(frames, 1024, device="cuda")
        ops.pool_score_save(h, frames, tokens, 1024, torch.ones(1024, device="cuda"), torch.zeros(1, device="cuda"), z, pooled)
        assert z.isnan().tolist() == [False, False, True, False, False] and (pooled[[0, 1, 3, 4]] - 1).abs().max() <= tokens * U32


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(ops):
    """the same operators on other data on two streams, without a wait in between: each result is its own"""
    from videoitg_amd.torch_ops import K
    steps = [Step(BF16, frames=40, tokens=9, k=256, f=192, vocab=300, seed=s) for s in (11, 12)]
    want = [{n: t.clone() for n, t in st.run(K).items()} for st in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (st, stream) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(stream):
                got[i] = st.run(K)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for n in w:
            assert torch.equal(w[n], g[n]), n


@pytest.mark.gpu
def test_dispatcher_forms_equal_the_binding(ops):
    from videoitg_amd.torch_ops import K
    grads = [randn(4000, dtype=F16, seed=1).cuda(), randn(33, seed=2).cuda()]
    outs, want = [torch.empty_like(t) for t in grads], [torch.empty_like(t) for t in grads]
    norm = K.clip_grad_norm(grads, 0.5, outs=outs, scale=0.5)
    assert torch.equal(norm, ops.clip_grad_norm(grads, 0.5, outs=want, scale=0.5)) and all(torch.equal(a, b) for a, b in zip(outs, want))
    assert torch.equal(K.clip_grad_norm(grads, None), ops.clip_grad_norm(grads, None))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        z = torch.empty(7, device="cuda")
        loss, weight, dz = torch.ops.videoitg.bce_loss_backward(z, z)
        assert loss.shape == () and weight.shape == () and dz.shape == (7,)
        assert torch.ops.videoitg.grad_norm([z]).shape == (1,)
    with pytest.raises(NotImplementedError):
        torch.ops.videoitg.embed_lookup(torch.zeros(1, dtype=torch.int64), torch.zeros(2, 4), torch.zeros(1, 4))


# ---- refusals ------------------------------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    from videoitg_amd import _lib
    return _lib.load()


P, ODD = C.c_void_p(4096), C.c_void_p(4098)        # addresses that nothing looks at: every call below is refused on the host
NUL = C.c_void_p(0)
SHAPE, ALIGN, DTYPE, ARG = -1, -2, -3, -4


def test_embed_entries_refuse(lib):
    def lookup(n=4, tdt=1, ldt=8, vocab=10, d=8, out=P, odt=2, ldo=8, ids=P, table=P):
        return lib.vitg_embed_lookup(ids, n, table, tdt, ldt, vocab, d, 1.0, out, odt, ldo, NUL)
    assert lookup(n=0, ids=NUL) == 0
    assert lookup(ids=NUL) == ARG and lookup(table=NUL) == ARG and lookup(out=NUL) == ARG
    assert lookup(tdt=3) == DTYPE and lookup(odt=-1) == DTYPE
    assert lookup(vocab=0) == SHAPE and lookup(ldt=4) == SHAPE and lookup(ldo=4) == SHAPE and lookup(d=0) == SHAPE and lookup(n=1 << 31) == SHAPE
    assert lookup(d=6, ldt=8) == ALIGN and lookup(ldt=10) == ALIGN and lookup(out=ODD) == ALIGN and lookup(table=ODD) == ALIGN

    need = C.c_long(-1)
    assert lib.vitg_embed_backward_plan(0, 8, C.byref(need)) == 0 and need.value == 0
    assert lib.vitg_embed_backward_plan(100, 8, C.byref(need)) == 0 and need.value > 100 * 16
    assert lib.vitg_embed_backward_plan((1 << 24) + 1, 8, C.byref(need)) == SHAPE and lib.vitg_embed_backward_plan(1 << 24, 8, C.byref(need)) == 0
    assert lib.vitg_embed_backward_plan(-1, 8, C.byref(need)) == SHAPE and lib.vitg_embed_backward_plan(4, 8, None) == ARG
    assert lib.vitg_embed_backward_plan(4, 8, C.byref(need)) == 0

    def back(n=4, ddt=1, ldd=8, vocab=10, d=8, tdt=2, ldt=8, ws=P, bytes_=need.value, ids=P, dout=P, table=P):
        return lib.vitg_embed_backward(ids, n, dout, ddt, ldd, vocab, d, 1.0, table, tdt, ldt, 0, ws, bytes_, NUL)
    assert back(table=NUL) == ARG and back(ids=NUL) == ARG and back(dout=NUL) == ARG and back(ws=NUL) == ARG and back(bytes_=need.value - 1) == ARG
    assert back(ddt=7) == DTYPE and back(tdt=7) == DTYPE
    assert back(n=(1 << 24) + 1) == SHAPE
    assert back(n=-1) == SHAPE and back(vocab=0) == SHAPE and back(ldd=4) == SHAPE and back(ldt=4) == SHAPE and back(vocab=1 << 31) == SHAPE
    assert back(d=6) == ALIGN and back(ldd=10) == ALIGN and back(ldt=10) == ALIGN and back(table=ODD) == ALIGN and back(dout=ODD) == ALIGN and back(ws=ODD) == ARG


def test_swiglu_entries_refuse(lib):
    def fwd(x=P, ldx=64, w=P, ldw=64, m=4, n=128, k=64, dt=1, out=P, ldo=64, gu=P, ldgu=128):
        return lib.vitg_swiglu(x, ldx, w, ldw, m, n, k, dt, out, ldo, gu, ldgu, NUL)
    assert fwd(m=0, x=NUL) == 0
    assert fwd(x=NUL) == ARG and fwd(w=NUL) == ARG and fwd(out=NUL) == ARG
    assert fwd(dt=2) == DTYPE
    assert fwd(k=32) == SHAPE and fwd(n=96) == SHAPE and fwd(ldx=56) == SHAPE and fwd(ldo=56) == SHAPE and fwd(ldgu=120) == SHAPE and fwd(ldw=1 << 22) == SHAPE
    assert fwd(m=(1 << 31) - 1) == SHAPE and fwd(n=1 << 30, ldo=1 << 29, ldgu=1 << 30) == SHAPE
    assert fwd(ldx=68) == ALIGN and fwd(ldgu=132) == ALIGN and fwd(x=ODD) == ALIGN and fwd(gu=ODD) == ALIGN

    need = C.c_long(-1)
    assert lib.vitg_swiglu_backward_plan(4, 128, 64, 1, 1, C.byref(need)) == 0 and need.value > 0
    assert lib.vitg_swiglu_backward_plan(4, 100, 64, 1, 1, C.byref(C.c_long(0))) == SHAPE and lib.vitg_swiglu_backward_plan(4, 128, 64, 1, 1, None) == ARG

    def back(dout=P, lddo=64, gu=P, ldgu=128, x=P, ldx=64, w=P, ldw=64, m=4, n=128, k=64, dt=1, dx=P, lddx=64, dw=P, lddw=64, dwdt=1, ws=P, bytes_=need.value):
        return lib.vitg_swiglu_backward(dout, lddo, gu, ldgu, x, ldx, w, ldw, m, n, k, dt, dx, lddx, dw, lddw, dwdt, 0, ws, bytes_, NUL)
    assert back(dx=NUL, dw=NUL) == 0
    assert back(dout=NUL) == ARG and back(gu=NUL) == ARG and back(x=NUL) == ARG and back(w=NUL) == ARG and back(ws=NUL) == ARG and back(bytes_=need.value - 1) == ARG
    assert back(dt=2) == DTYPE and back(dwdt=0) == DTYPE
    assert back(n=96) == SHAPE and back(k=60) == SHAPE and back(m=-1) == SHAPE and back(lddx=56) == SHAPE and back(lddw=56) == SHAPE and back(m=1 << 22) == SHAPE
    assert back(lddo=68) == ALIGN and back(lddw=68) == ALIGN and back(dw=ODD) == ALIGN and back(dx=ODD) == ALIGN


def test_head_and_clip_entries_refuse(lib):
    def save(h=P, dt=2, ldh=8, frames=2, tokens=3, d=8, w=P, b=P, logits=P, pooled=P, ldp=8):
        return lib.vitg_pool_score_save(h, dt, ldh, frames, tokens, d, w, b, logits, pooled, ldp, NUL)
    assert save(frames=0, h=NUL) == 0
    assert save(h=NUL) == ARG and save(pooled=NUL) == ARG and save(dt=5) == DTYPE and save(tokens=0) == SHAPE and save(ldh=4) == SHAPE
    assert save(frames=1 << 22) == SHAPE
    assert save(d=6) == ALIGN and save(w=ODD) == ALIGN and save(ldp=10) == ALIGN
    assert lib.vitg_bce_loss_backward(P, P, 0, 1.0, P, P, NUL) == ARG and lib.vitg_bce_loss_backward(P, P, 3, 1.0, P, NUL, NUL) == ARG

    def back(pooled=P, ldp=8, frames=2, tokens=3, d=8, w=P, dz=P, dh=P, dt=2, lddh=8, dw=P, db=P):
        return lib.vitg_pool_score_backward(pooled, ldp, frames, tokens, d, w, dz, dh, dt, lddh, dw, db, 0, NUL)
    assert back(dh=NUL, dw=NUL, db=NUL) == 0
    assert back(pooled=NUL) == ARG and back(w=NUL) == ARG and back(dz=NUL) == ARG and back(dt=4) == DTYPE and back(tokens=0) == SHAPE and back(frames=-1) == SHAPE
    assert back(frames=1 << 24, tokens=1) == SHAPE and back(frames=1, tokens=(1 << 31) - 1, dw=NUL, db=NUL) == SHAPE
    assert back(lddh=4) == SHAPE and back(ldp=4) == SHAPE and back(d=6) == ALIGN and back(dh=ODD) == ALIGN

    one, f32 = (C.c_long * 1)(5), (C.c_int * 1)(2)
    ptr, odd, nul = (C.c_void_p * 1)(4096), (C.c_void_p * 1)(4098), (C.c_void_p * 1)(0)
    need = C.c_long(0)
    assert lib.vitg_clip_grad_plan(1, one, f32, C.byref(need)) == 0 and need.value >= 8
    assert lib.vitg_clip_grad_plan(-1, one, f32, C.byref(need)) == SHAPE and lib.vitg_clip_grad_plan(1, (C.c_long * 1)(-1), f32, C.byref(need)) == SHAPE
    assert lib.vitg_clip_grad_plan(1, one, (C.c_int * 1)(9), C.byref(need)) == DTYPE

    far = C.c_void_p(1 << 20)

    def clip(count=1, g=ptr, o=ptr, numel=one, dt=f32, max_norm=1.0, norm=C.c_void_p(1 << 16), ws=far, bytes_=64):
        return lib.vitg_clip_grad(count, g, o, numel, dt, 1.0, max_norm, norm, ws, bytes_, NUL)
    assert clip(g=nul) == ARG and clip(o=nul) == ARG and clip(norm=NUL) == ARG and clip(ws=NUL) == ARG and clip(bytes_=4) == ARG and clip(max_norm=-1.0) == ARG
    both, five, kinds = C.c_void_p * 2, (C.c_long * 2)(5, 5), (C.c_int * 2)(2, 2)
    for g, o in (((4096, 4096), (4096, 4096)), ((4096, 4112), (4096, 4112)), ((4096, 8192), (8192, 12288)), ((4096, 8192), (12288, 12300)), ((4096, 8192), (4100, 8192))):
        assert clip(count=2, g=both(*g), o=both(*o), numel=five, dt=kinds) == ARG, (g, o)        # two tensors on one byte that is written
    assert clip(norm=C.c_void_p(4100)) == ARG and clip(ws=P) == ARG
    assert clip(max_norm=float("nan")) == ARG and clip(g=odd) == ALIGN and clip(dt=(C.c_int * 1)(3)) == DTYPE and clip(count=-1) == SHAPE


def test_wrappers_refuse_host_tensors():
    from videoitg_amd import ops
    from videoitg_amd._lib import VitgError
    x = torch.zeros(4, 64, dtype=F16)
    for call in (lambda: ops.embed_lookup(torch.zeros(4, dtype=torch.int64), x, x), lambda: ops.swiglu(x, x, x), lambda: ops.clip_grad_norm([x], 1.0),
                 lambda: ops.clip_grad_norm([], 1.0), lambda: ops.bce_loss_backward(x[0], x[0])):
        with pytest.raises(VitgError):
            call()


@pytest.mark.gpu
def test_wrappers_refuse(ops):
    from videoitg_amd._lib import VitgError
    z = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device="cuda")            # noqa: E731
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    x, w = z(4, 64, dt=F16), z(128, 64, dt=F16)
    gu, out = z(4, 128, dt=F16), z(4, 64, dt=F16)
    big = z(6, 8)
    calls = {
        "ids of another type": lambda: ops.embed_lookup(ids.int(), z(5, 8), z(4, 8)),
        "too few output rows": lambda: ops.embed_lookup(ids, z(5, 8), z(3, 8)),
        "transposed output": lambda: ops.embed_lookup(ids, z(5, 8), z(8, 4).t()),
        "rows that overlap": lambda: ops.embed_backward(ids, z(4, 8), torch.as_strided(z(64), (5, 8), (4, 1))),
        "expanded rows": lambda: ops.embed_backward(ids, z(4, 8), z(1, 8).expand(5, 8)),
        "output on the table": lambda: ops.embed_lookup(ids, big, big[:4]),
        "width no multiple of four": lambda: ops.embed_lookup(ids, z(5, 6), z(4, 6)),
        "integer table": lambda: ops.embed_lookup(ids, ids.view(2, 2), z(4, 2)),
        "a short workspace": lambda: ops.embed_backward(ids, z(4, 8), z(5, 8), workspace=z(4)),
        "a workspace on the gradient": lambda: ops.embed_backward(ids, z(4, 8), big, workspace=torch.as_strided(big, (48,), (1,)).view(torch.uint8)),
        "weights of another type": lambda: ops.swiglu(x, w.bfloat16(), out),
        "fp32 activations": lambda: ops.swiglu(x.float(), w.float(), out.float()),
        "an inner width of 96": lambda: ops.swiglu(z(4, 96, dt=F16), z(128, 96, dt=F16), out),
        "pre-activations on the output": lambda: ops.swiglu(x, w, gu[:, :64], gu=gu),
        "pre-activations too narrow": lambda: ops.swiglu(x, w, out, gu=gu[:, :64]),
        "gradient over its input": lambda: ops.swiglu_backward(out, gu, x, w, dx=x),
        "one buffer for both gradients": lambda: ops.swiglu_backward(out, gu, x, w, dx=gu.view(8, 64)[:4], dw=w),
        "weight gradient of a third type": lambda: ops.swiglu_backward(out, gu, x, w, dw=w.bfloat16()),
        "weight gradient in 64 bits": lambda: ops.swiglu_backward(out, gu, x, w, dw=w.double()),
        "no tokens per frame": lambda: ops.pool_score_save(z(4, 8), 4, 0, 8, z(8), z(1), z(4), z(4, 8)),
        "labels of another length": lambda: ops.bce_loss_backward(z(4), z(5)),
        "no frames": lambda: ops.bce_loss_backward(z(0), z(0)),
        "head weights in 16 bits": lambda: ops.pool_score_backward(z(4, 8), 4, 1, 8, z(8, dt=F16), z(4), z(4, 8)),
        "a gradient that is no contiguous tensor": lambda: ops.clip_grad_norm([z(8, 8).t()[:3]], 1.0),
        "the same tensor twice in place": lambda: ops.clip_grad_norm([big, big], 1.0),
        "overlapping views": lambda: ops.clip_grad_norm([big[:4], big[3:]], 1.0),
        "an output on another gradient": lambda: ops.clip_grad_norm([big[:3], big[3:]], 1.0, outs=[big[3:], z(3, 8)]),
        "an output of another type": lambda: ops.clip_grad_norm([big], 1.0, outs=[big.half()]),
        "fewer outputs": lambda: ops.clip_grad_norm([big, z(3)], 1.0, outs=[big]),
        "a negative limit": lambda: ops.clip_grad_norm([big], -1.0),
        "integer gradients": lambda: ops.clip_grad_norm([ids], 1.0),
        "outputs without a limit": lambda: ops.clip_grad_norm([big], None, outs=[z(6, 8)]),
    }
    for what, call in calls.items():
        with pytest.raises(VitgError):
            call()
            pytest.fail(what)
    # and what is allowed: the same tensor twice where nothing is written
    assert ops.clip_grad_norm([z(2) + 1, z(2) + 1], None).item() == 2.0
    twice = z(2) + 1
    assert ops.clip_grad_norm([twice, twice], None).item() == 2.0
