"""The training operators at their edges: what the documentation allows and tests/test_train_ops.py does not call."""
import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs an MI355X"
    from videoitg_amd import ops as o
    return o


def interleave(gate, up):
    return torch.stack([gate.unflatten(-1, (-1, 32)), up.unflatten(-1, (-1, 32))], -2).flatten(-3)


# rows few enough for one pass; ring kernel with a join; 256x256 tiles whole, with ragged edges too; tiles split over the rows; 256x384 tiles whole
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [(20, 1088, 2048), (300, 256, 832), (2100, 1024, 16384), (1100, 1088, 16448), (7000, 1088, 2048), (4100, 3584, 9472)])
def test_weight_gradient_is_added_once_on_every_route(ops, dtype, m, k, n):
    """gate = 0 (sigmoid 1/2, dU = 0), up 1 or 2 and whole x and dout: dGU and every partial sum are exact, so that one rounding is left - that of old + sum.  A route
    that carries the large old value through the sum rounds once per step"""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    whole = lambda *s: torch.randint(-4, 5, s, generator=g, device="cuda", dtype=torch.int32).to(dtype)      # noqa: E731
    x, dout, w = whole(m, k), whole(m, n // 2), whole(n, k)
    up = torch.randint(1, 3, (m, n // 2), generator=g, device="cuda").to(dtype)
    gu = interleave(torch.zeros_like(up), up)
    old = torch.randn(n, k, generator=g, device="cuda") * 1e5
    dgu = interleave(dout.double() * up.double() / 2, torch.zeros_like(up, dtype=torch.float64))
    want = (old.double() + dgu.t() @ x.double()).float()
    for dx in (None, torch.empty_like(x)):
        dw = old.clone()
        ops.swiglu_backward(dout, gu, x, w, dx=dx, dw=dw, accumulate=True)
        assert torch.equal(dw, want), f"{int((dw != want).sum())} of {dw.numel()} rounded more than once"


@pytest.mark.gpu
def test_loss_of_the_most_logits_a_call_takes(ops):
    """2^31 - 1 logits and frames: an index that wraps behind the last one reads and writes outside.  All logits 0 but the last few, so that everything is known"""
    n = (1 << 31) - 1
    z, y = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    z[-3:] = torch.tensor([40.0, -40.0, 2.0], device="cuda")
    y[:1 << 30] = 1.0                                    # one label more than none of them: pos_weight = sqrt((2^30 - 1) / 2^30), 1 in fp32
    loss, weight, dz = ops.bce_loss_backward(z, y, scale=float(1 << 31))
    assert weight.item() == 1.0
    assert abs(loss.item() / 0.6931471805599453 - 1) <= 2.0 ** -20
    assert (dz[:1 << 30] == -0.5).all() and (dz[1 << 30:-3] == 0.5).all()
    want = torch.sigmoid(torch.tensor([40.0, -40.0, 2.0], dtype=torch.float64))
    assert ((dz[-3:].double().cpu() - want).abs() <= want * 2.0 ** -20).all()
    plain, weight = ops.bce_loss(z, y)
    assert weight.item() == 1.0 and 0.5 < plain.item() < 0.9      # (2^21 fp32 terms a thread, rounded at up to 2^21)
    db = torch.zeros(1, device="cuda")
    ops.pool_score_backward(torch.empty(n, 4, device="cuda"), n, 1, 4, torch.ones(4, device="cuda"), dz, db=db)
    assert abs(db.item() - (want.sum().item() - 2.0)) <= 1e-6
    del z, y, dz
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_head_gradient_of_the_widest_rows(ops):
    """rows of 2^31 - 8 values: the last step past a row must not wrap either"""
    d = (1 << 31) - 8
    w = torch.zeros(d, device="cuda")
    w[-8:] = torch.arange(1.0, 9.0, device="cuda")
    w[:4] = 3.0
    dh = torch.full((2, d), 7.0, dtype=F16, device="cuda")
    ops.pool_score_backward(torch.empty(2, d, device="cuda"), 2, 1, d, w, torch.tensor([1.0, -2.0], device="cuda"), dh)
    for row, z in enumerate((1.0, -2.0)):
        assert (dh[row, :4] == 3.0 * z).all() and (dh[row, 4:-8] == 0).all() and (dh[row, -8:] == z * w[-8:]).all()
    del w, dh
    torch.cuda.empty_cache()


def test_dispatcher_form_of_clipping_refuses_what_the_binding_refuses():
    from videoitg_amd._lib import VitgError
    from videoitg_amd.torch_ops import K
    g = [torch.ones(3)]
    for call in (lambda: K.clip_grad_norm(g, None, outs=[torch.zeros(3)]), lambda: K.clip_grad_norm([], 1.0), lambda: K.clip_grad_norm(iter(()), None)):
        with pytest.raises(VitgError):
            call()


@pytest.mark.gpu
def test_dispatcher_form_of_clipping_takes_every_argument(ops):
    from videoitg_amd.torch_ops import K
    make = lambda: [torch.arange(1.0, 3000.0, device="cuda").to(F16), torch.arange(7.0, device="cuda")]      # noqa: E731
    zeros = lambda: [torch.zeros_like(t) for t in make()]                                                     # noqa: E731
    with pytest.raises(Exception, match="no outs"):
        K.clip_grad_norm(make(), None, outs=zeros())
    with pytest.raises(Exception, match="no outs"):
        torch.ops.videoitg.clip_grad_norm_into(make(), zeros(), torch.zeros(1, device="cuda"), None)
    with pytest.raises(Exception, match="2 gradients and 0 outputs"):
        torch.ops.videoitg.clip_grad_norm_into(make(), [], torch.zeros(1, device="cuda"), 1.0)
    ws = torch.empty(4096, dtype=torch.uint8, device="cuda")
    for max_norm in (0.5, None):
        for outs in (False, True):
            if outs and max_norm is None:
                continue
            for norm in (False, True):
                for workspace in (None, ws):
                    got, want, o, p = make(), make(), zeros(), zeros()
                    slot = torch.full((1,), -1.0, device="cuda") if norm else None
                    a = K.clip_grad_norm(iter(got), max_norm, outs=iter(o) if outs else None, scale=0.25, norm=slot, workspace=workspace)
                    b = ops.clip_grad_norm(want, max_norm, outs=p if outs else None, scale=0.25)
                    assert torch.equal(a, b) and (not norm or a is slot)
                    assert all(torch.equal(x, y) for x, y in zip(got + o, want + p))


def shifted(t, ld=0):
    """the same values 16 bytes behind a 32-byte boundary, rows `ld` apart"""
    rows, cols = t.shape if t.dim() == 2 else (1, t.numel())
    ld = max(ld, cols)
    flat = torch.zeros(rows * ld + 64, dtype=t.dtype, device="cuda")
    assert flat.data_ptr() % 32 == 0
    out = torch.as_strided(flat, (rows, cols), (ld, 1), 16 // t.element_size())
    out.copy_(t.view(rows, cols))
    return out if t.dim() == 2 else out[0]


@pytest.mark.gpu
@pytest.mark.parametrize("half", [BF16, F16])
def test_fp32_operands_16_bytes_behind_a_32_byte_boundary(ops, half):
    """eight values of a lane are two 16-byte accesses: 16-byte aligned rows of fp32 give the bits of fully aligned ones"""
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s, dtype=F32: torch.randn(*s, generator=g, device="cuda").to(dtype)      # noqa: E731
    ids = torch.randint(-1, 40, (300,), generator=g, device="cuda")
    table, dout = rand(40, 264), rand(300, 264)
    for dtype in (half, F32):
        same = ops.embed_lookup(ids, shifted(table), shifted(torch.zeros(300, 264, dtype=dtype)))
        assert torch.equal(same, ops.embed_lookup(ids, table, torch.zeros(300, 264, dtype=dtype, device="cuda")))
        for add in (False, True):
            a, b = shifted(table.to(dtype)), table.to(dtype)
            ops.embed_backward(ids, shifted(dout), a, accumulate=add)
            ops.embed_backward(ids, dout, b, accumulate=add)
            assert torch.equal(a, b)
    x, gu, up = rand(20, 128, dtype=half), rand(20, 256, dtype=half), rand(20, 128, dtype=half)
    a, b = shifted(torch.ones(256, 128)), torch.ones(256, 128, device="cuda")
    w = rand(256, 128, dtype=half)
    ops.swiglu_backward(up, gu, x, w, dw=a, accumulate=True)
    ops.swiglu_backward(up, gu, x, w, dw=b, accumulate=True)
    assert torch.equal(a, b)
    for frames, tokens in ((9, 5), (3, 150)):            # one block a frame; rows over several blocks
        h, hw, bias = rand(frames * tokens, 520, dtype=half), rand(520), rand(1)
        z, zs, p, ps = (torch.empty(frames, device="cuda"), torch.empty(frames, device="cuda"), torch.empty(frames, 520, device="cuda"), shifted(torch.zeros(frames, 520), 524))
        ops.pool_score_save(h, frames, tokens, 520, hw, bias, z, p)
        ops.pool_score_save(h, frames, tokens, 520, shifted(hw), bias, zs, ps)
        assert torch.equal(z, zs) and torch.equal(p, ps)
        d, ds, dw, dws = torch.empty_like(h), torch.empty_like(h), torch.empty_like(hw), shifted(torch.zeros(520))
        ops.pool_score_backward(p, frames, tokens, 520, hw, z, d, dw=dw)
        ops.pool_score_backward(ps, frames, tokens, 520, shifted(hw), z, ds, dw=dws)
        assert torch.equal(d, ds) and torch.equal(dw, dws)
    t = shifted(rand(70000))
    u = t.clone()
    assert torch.equal(ops.clip_grad_norm([t], 1.0), ops.clip_grad_norm([u], 1.0)) and torch.equal(t, u)


def test_shared_memory_is_found_byte_for_byte():
    """every pair of row blocks in a small buffer against the sets of bytes they hold; only rows of two pitches may be refused without need"""
    from videoitg_amd import ops
    checked = refused = 0
    flat = torch.zeros(96, dtype=F16)
    views = [torch.as_strided(flat, (rows, cols), (ld, 1), at) for rows in (1, 2, 3) for ld in (8, 12) for cols in (2, 5, 8, 12) if cols <= ld for at in (0, 1, 3, 7, 8, 13, 24, 30)
             if at + (rows - 1) * ld + cols <= 96]
    held = [{v.storage_offset() + i * v.stride(0) + j for i in range(v.shape[0]) for j in range(v.shape[1])} for v in views]
    item = lambda v: ("v", v.data_ptr(), v.data_ptr() + 2 * ((v.shape[0] - 1) * v.stride(0) + v.shape[1]), v)      # noqa: E731
    items = [item(v) for v in views]
    for v, p, a in zip(views, items, held):
        for u, q, b in zip(views, items, held):
            meet = ops._meet(p, q)
            if a & b:
                assert meet
            elif meet:
                assert v.shape[0] > 1 and u.shape[0] > 1 and v.stride(0) != u.stride(0)
                refused += 1
            checked += 1
    assert checked > 5000 and refused < checked / 10
    assert not ops._meet(("empty", 100, 100), ("v", 50, 150)) and ops._meet(("a", 100, 120), ("b", 119, 130)) and not ops._meet(("a", 100, 120), ("b", 120, 130))


@pytest.mark.gpu
def test_column_slices_of_one_buffer(ops):
    """operands and results side by side in one buffer give the bits of separate ones; slices that share a column are refused"""
    from videoitg_amd._lib import VitgError
    g = torch.Generator(device="cuda").manual_seed(8)
    rand = lambda *s, dtype=F32: torch.randn(*s, generator=g, device="cuda").to(dtype)      # noqa: E731
    for m, k, n in ((9, 128, 192), (70, 64, 320), (300, 256, 832), (600, 1024, 128)):
        x, w, dout = rand(m, k, dtype=BF16), rand(n, k, dtype=BF16), rand(m, n // 2, dtype=BF16)
        act, gu, dx, dw = x.new_empty(m, n // 2), x.new_empty(m, n), torch.empty_like(x), torch.empty_like(w)
        ops.swiglu(x, w, act, gu=gu)
        ops.swiglu_backward(dout, gu, x, w, dx=dx, dw=dw)
        rows = torch.full((m, 2 * k + 2 * n), 7.0, dtype=BF16, device="cuda")
        xs, acts, gus, dxs, douts = rows.split([k, n // 2, n, k, n // 2], 1)
        both = torch.full((n, 2 * k), 7.0, dtype=BF16, device="cuda")
        ws, dws = both.split(k, 1)
        xs.copy_(x), douts.copy_(dout), ws.copy_(w)
        ops.swiglu(xs, ws, acts, gu=gus)
        ops.swiglu_backward(douts, gus, xs, ws, dx=dxs, dw=dws)
        for got, want in ((acts, act), (gus, gu), (dxs, dx), (dws, dw), (xs, x), (ws, w), (douts, dout)):
            assert torch.equal(got, want)
        with pytest.raises(VitgError, match="share memory"):
            ops.swiglu(xs, ws, rows[:, k - 8:k - 8 + n // 2])
    ids = torch.randint(-1, 50, (400,), generator=g, device="cuda")
    one = rand(50, 2 * 96)
    table, dtable = one.split(96, 1)
    rows = rand(50, 2 * 96)[torch.arange(400, device="cuda") % 50]
    out, dout = rows.split(96, 1)
    want = ops.embed_lookup(ids, table.contiguous(), torch.empty(400, 96, device="cuda"))
    grad = ops.embed_backward(ids, dout.contiguous(), torch.empty(50, 96, device="cuda"))
    assert torch.equal(ops.embed_lookup(ids, table, out), want) and torch.equal(ops.embed_backward(ids, dout, dtable), grad)
    h = rand(60 * 5, 2 * 264)
    w, b, z, z2, pooled = rand(264), rand(1), torch.empty(60, device="cuda"), torch.empty(60, device="cuda"), torch.empty(60, 264, device="cuda")
    ops.pool_score_save(h[:, :264].contiguous(), 60, 5, 264, w, b, z, pooled)
    ops.pool_score_save(h[:, :264], 60, 5, 264, w, b, z2, pooled)
    dh = torch.empty(300, 264, device="cuda")
    ops.pool_score_backward(pooled, 60, 5, 264, w, z, dh)
    ops.pool_score_backward(pooled, 60, 5, 264, w, z2, h[:, 264:])
    assert torch.equal(z, z2) and torch.equal(h[:, 264:], dh)


@pytest.mark.gpu
@pytest.mark.parametrize("low,high", [(3.0, 6.0), (9.0, 11.0), (14.0, 30.0), (60.0, 90.0)])
def test_loss_of_scores_that_are_right(ops, low, high):
    """every frame on its own side: the loss is a sum of exponentials.  A term is off by the rounding of the logarithm (2 units), the exponential (2 units; its argument is exact),
    a product and two sums, half a unit of 2^-23 each, the weight by 3 units: 2^-20 together"""
    g = torch.Generator().manual_seed(int(low))
    y = (torch.rand(700, generator=g) < 0.3).float()
    z = (torch.rand(700, generator=g) * (high - low) + low) * (2 * y - 1)
    z64, y64 = z.double(), y.double()
    pos = float(y64.sum())
    pw = min(5.0, ((700 - pos) / max(1.0, pos)) ** 0.5)
    want = -(pw * y64 * torch.nn.functional.logsigmoid(z64) + (1 - y64) * torch.nn.functional.logsigmoid(-z64)).mean().item()
    loss, weight, dz = ops.bce_loss_backward(z.cuda(), y.cuda())
    assert abs(loss.item() / want - 1) <= 2.0 ** -20


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 1e-12, 1e-30])
def test_clipping_by_a_factor_below_the_normal_numbers(ops, max_norm):
    """norms of 1e39 and more: the factor has no fp32 value of 24 bits, the results do"""
    g = torch.Generator().manual_seed(4)
    grads = [(torch.rand(3000, generator=g) + 0.1) * 3e38, ((torch.rand(517, generator=g) + 0.1) * 3e38).to(BF16), torch.randn(5, generator=g) * 1e30, torch.full((3,), -1e20)]
    limit = float(torch.tensor(max_norm, dtype=F32))
    norm = sum(float(t.double().square().sum()) for t in grads) ** 0.5
    assert limit / norm < 1.2e-38
    dev = [t.cuda() for t in grads]
    assert ops.clip_grad_norm(dev, max_norm).item() == float("inf")       # (beyond fp32)
    for t, o in zip(grads, dev):
        want = t.double() * (limit / (norm + 1e-6))
        half, least = (2.0 ** -8, 2.0 ** -133) if t.dtype == BF16 else (2.0 ** -24, 2.0 ** -149)
        bound = want.abs() * (4 * 2.0 ** -24 + half * 1.001) + least
        assert ((o.double().cpu() - want).abs() <= bound).all()
