"""moe_permute / moe_unpermute and their gradients against the definition in 64 bits.

What only moves is compared bit for bit.  A weighted sum of n terms in fp32 is off by at most (n + 1) * 2^-24 of the sum of
its terms' absolute values (n products or additions fused, the first from zero), and by half a step of the output
type for the cast.
"""
import pytest
import torch
from torch.autograd import forward_ad

import flag_gems
from flaggems_b200 import _cabi

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
FLOATS = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ids(t, e, k, g, dtype=torch.int32):
    """Distinct experts where there are enough, any otherwise."""
    if k <= e:
        return torch.rand(t, e, device="cuda", generator=g).topk(k, 1).indices.to(dtype)
    return torch.randint(0, e, (t, k), device="cuda", generator=g).to(dtype)


def _plan(ids, e, expert_map=None):
    flat = ids.reshape(-1).long()
    if expert_map is not None:
        known = (flat >= 0) & (flat < expert_map.numel())
        flat = torch.where(known, expert_map.long()[flat.clamp(0, expert_map.numel() - 1)], -1)
    bucket = torch.where((flat >= 0) & (flat < e), flat, e)
    slot_of_row = torch.argsort(bucket, stable=True)
    row_of_slot = torch.empty_like(slot_of_row)
    row_of_slot[slot_of_row] = torch.arange(flat.numel(), device=flat.device)
    row_of_slot = torch.where(bucket < e, row_of_slot, -1 - row_of_slot)
    offs = torch.bincount(bucket, minlength=e + 1)[:e].cumsum(0)
    return offs.int(), row_of_slot.view(ids.shape).int(), slot_of_row.int()


def _same_plan(plan, want):
    for got, w in zip(plan, want):
        assert got.dtype == torch.int32 and got.is_contiguous() and torch.equal(got, w)


def _bytes(x):
    return x.contiguous().view(torch.uint8)


def _check_permuted(x, rows, plan, topk):
    valid = int(plan.offs[-1])
    src = (plan.slot_of_row // topk).long()
    assert torch.equal(_bytes(rows[:valid]), _bytes(x[src[:valid]]))
    assert not _bytes(rows[valid:]).any()


def _check_sum(got, rows, row_of_slot, w):
    t, k = row_of_slot.shape
    r = row_of_slot.clamp_min(0).long()
    real = (row_of_slot >= 0)[:, :, None]
    prod = torch.where(real, rows[r].double(), 0.0)
    if w is not None:
        prod = prod * torch.where(real[:, :, 0], w.double(), 0.0)[:, :, None]
    want, mass = prod.sum(1), prod.abs().sum(1)
    half = torch.finfo(got.dtype).eps / 2
    bound = mass * (k + 1) * F32 + want.abs() * half * (1 + 8 * F32) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert bool(((got.double() - want).abs() <= bound * 1.01 + mass * (k + 1) * F32 * half).all())


# tokens, experts per token, experts, hidden
SHAPES = [(1, 1, 1, 8), (1, 8, 256, 7168), (3, 2, 8, 40), (5, 3, 2, 16), (64, 8, 256, 7168), (33, 4, 1024, 64), (127, 6, 60, 520),
          (130, 1, 3, 4096), (515, 10, 319, 136), (1023, 2, 8, 2056), (2048, 8, 256, 64), (3000, 32, 64, 24), (9001, 8, 160, 16),
          (16384, 8, 256, 32), (70000, 2, 8, 16), (17, 2, 8, 7), (4, 2, 4, 1), (2, 1, 2, 20000), (300, 8, 33, 1000), (6, 40, 64, 72)]


@pytest.mark.parametrize("t,k,e,h", SHAPES)
@pytest.mark.parametrize("dtype", FLOATS + [torch.int8])
def test_permute(t, k, e, h, dtype):
    g = _gen(t + h)
    x = (torch.randn(t, h, device="cuda", generator=g) * 30).to(dtype)
    ids = _ids(t, e, k, g, torch.int64 if h % 3 == 0 else torch.int32)
    rows, scale, plan = flag_gems.moe_permute(x, ids, e)
    assert scale is None and rows.dtype == dtype and rows.shape == (t * k, h)
    _same_plan(plan, _plan(ids, e))
    _check_permuted(x, rows, plan, k)


@pytest.mark.parametrize("t,k,e,h", SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_unpermute(t, k, e, h, dtype):
    g = _gen(t + h)
    ids = _ids(t, e, k, g)
    plan = flag_gems.MoEPermutation(*_plan(ids, e))
    rows = torch.randn(t * k, h, device="cuda", generator=g).to(dtype)
    for w in (None, torch.randn(t, k, device="cuda", generator=g), torch.rand(t, k, device="cuda", generator=g).to(torch.bfloat16),
              torch.rand(t, k, device="cuda", generator=g).to(torch.float16)):
        out = flag_gems.moe_unpermute(rows, plan, w)
        assert out.shape == (t, h) and out.dtype == dtype
        _check_sum(out, rows, plan.row_of_slot, w)


@pytest.mark.parametrize("t,k,e,h", SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("w_dtype", [None, torch.float32, torch.bfloat16])
def test_gradients(t, k, e, h, dtype, w_dtype):
    g = _gen(t + h)
    ids = _ids(t, e, k, g)
    if t > 2:
        ids[1] = -1  # a token none of whose slots has an expert
        ids[2, 0] = e
    x = torch.randn(t, h, device="cuda", generator=g).to(dtype).requires_grad_()
    rows, _, plan = flag_gems.moe_permute(x, ids, e)
    d_rows = torch.randn(t * k, h, device="cuda", generator=g).to(dtype)
    d_rows[int(plan.offs[-1]):] = float("nan")  # gradients of rows without an expert are not read
    d_x, = torch.autograd.grad(rows, x, d_rows)
    assert d_x.dtype == dtype
    _check_sum(d_x, d_rows, plan.row_of_slot, None)

    y = torch.randn(t * k, h, device="cuda", generator=g).to(dtype)
    y[int(plan.offs[-1]):] = float("nan")
    y.requires_grad_()
    w = None if w_dtype is None else torch.randn(t, k, device="cuda", generator=g).to(w_dtype).requires_grad_()
    out = flag_gems.moe_unpermute(y, plan, w)
    _check_sum(out.detach(), y.detach(), plan.row_of_slot, None if w is None else w.detach())
    d_out = torch.randn(t, h, device="cuda", generator=g).to(dtype)
    d_y, *d_w = torch.autograd.grad(out, (y,) if w is None else (y, w), d_out)
    half = torch.finfo(dtype).eps / 2
    r = plan.row_of_slot.long()
    real = r >= 0
    tok = torch.arange(t, device="cuda")[:, None].expand(t, k)
    want = torch.zeros(t * k, h, dtype=torch.float64, device="cuda")
    want[r[real]] = d_out.double()[tok[real]] * (1.0 if w is None else w.detach().double()[real][:, None])
    err = (d_y.double() - want).abs()
    assert bool((err <= want.abs() * (half + 2 * F32) + (2.0 ** -25 if dtype == torch.float16 else 0.0)).all())
    if w is not None:
        prod = torch.zeros(t, k, h, dtype=torch.float64, device="cuda")
        prod[real] = y.detach().double()[r[real]] * d_out.double()[tok[real]]
        dot, mass = prod.sum(2), prod.abs().sum(2)
        # any order of h additions of products: (h + 1) * 2^-24, and the cast to the weights' type
        assert d_w[0].dtype == w_dtype and d_w[0].shape == (t, k)
        bound = mass * (h + 1) * F32 + dot.abs() * torch.finfo(w_dtype).eps / 2 * (1 + 2 * F32)
        assert bool(((d_w[0].double() - dot).abs() <= bound * 1.01).all())
        only_w, = torch.autograd.grad(flag_gems.moe_unpermute(y.detach(), plan, w), w, d_out)
        only_y, = torch.autograd.grad(flag_gems.moe_unpermute(y, plan, w.detach()), y, d_out)
        assert torch.equal(only_w, d_w[0]) and torch.equal(only_y, d_y)


def test_gradients_against_differences():
    """Both maps are linear in each argument: a central difference of step 1/2 is exact but for roundings."""
    g = _gen(3)
    t, k, e, h = 37, 3, 5, 24
    ids = torch.randint(-1, e + 1, (t, k), device="cuda", generator=g)
    x, w = torch.randn(t, h, device="cuda", generator=g), torch.randn(t, k, device="cuda", generator=g)
    a, b = torch.randn(t * k, h, device="cuda", generator=g), torch.randn(t, h, device="cuda", generator=g)

    def value(x, w):
        rows, _, plan = flag_gems.moe_permute(x, ids, e)
        return flag_gems.moe_unpermute(rows * a, plan, w), rows

    x_, w_ = x.clone().requires_grad_(), w.clone().requires_grad_()
    d_x, d_w = torch.autograd.grad((value(x_, w_)[0] * b).sum(), (x_, w_))
    for arg, grad in ((0, d_x), (1, d_w)):
        step = torch.randn(grad.shape, device="cuda", generator=g)
        hi, lo = ((value(x + s * step, w) if arg == 0 else value(x, w + s * step))[0].double() for s in (0.5, -0.5))
        diff = ((hi - lo) * b.double()).sum()
        mass = ((hi.abs() + lo.abs()) * b.double().abs()).sum() + (grad.double() * step.double()).abs().sum()
        assert abs(float(diff - (grad.double() * step.double()).sum())) <= float(mass) * 16 * F32


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [1, 56, 300])
def test_permute_with_scales(dtype, cols):
    g = _gen(cols)
    t, k, e, h = 77, 4, 9, 112
    x = (torch.randn(t, h, device="cuda", generator=g) * 20).to(dtype)
    scale = torch.rand(t, cols, device="cuda", generator=g)
    ids = _ids(t, e, k, g)
    ids[5:9] = -7
    for s in (scale, scale.t().contiguous().t(), torch.cat([scale, scale], 1)[:, :cols]):
        rows, row_scale, plan = flag_gems.moe_permute(x, ids, e, scale=s)
        _same_plan(plan, _plan(ids, e))
        _check_permuted(x, rows, plan, k)
        valid = int(plan.offs[-1])
        assert valid == t * k - 16
        assert torch.equal(row_scale[:valid], scale[(plan.slot_of_row // k).long()][:valid])
        assert bool((row_scale[valid:] == 1.0).all())


@pytest.mark.parametrize("t", [1, 300, 5000])
def test_slots_without_an_expert(t):
    g = _gen(t)
    k, e, h = 8, 32, 128
    x = torch.randn(t, h, device="cuda", generator=g).bfloat16()
    ids = torch.randint(-3, 300, (t, k), device="cuda", generator=g)
    ids[0, 0] = 2 ** 40  # past 32 bits
    _same_plan(flag_gems.moe_permute(x, ids, e)[2], _plan(ids, e))
    # a rank that holds 32 of 256 experts
    expert_map = torch.full((256,), -1, dtype=torch.int64, device="cuda")
    expert_map[64:96] = torch.arange(32, device="cuda").flip(0)
    rows, _, plan = flag_gems.moe_permute(x, ids, e, expert_map=expert_map)
    _same_plan(plan, _plan(ids, e, expert_map))
    _check_permuted(x, rows, plan, k)
    none = torch.full((t, k), -1, dtype=torch.int32, device="cuda")
    rows, _, plan = flag_gems.moe_permute(x, none, e)
    assert not rows.any() and not plan.offs.any() and bool((plan.row_of_slot < 0).all())
    junk = torch.full((t * k, h), float("nan"), device="cuda")
    assert not flag_gems.moe_unpermute(junk, plan, torch.full((t, k), float("inf"), device="cuda")).any()


def test_one_expert_takes_all():
    x = torch.randn(5000, 64, device="cuda", generator=_gen())
    ids = torch.full((5000, 2), 7, dtype=torch.int32, device="cuda")  # the same expert twice
    rows, _, plan = flag_gems.moe_permute(x, ids, 9)
    _same_plan(plan, _plan(ids, 9))
    assert torch.equal(rows, x.repeat_interleave(2, 0))
    assert torch.equal(flag_gems.moe_unpermute(rows, plan), x + x)


def test_nothing_to_move():
    ids = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    rows, _, plan = flag_gems.moe_permute(x, ids, 6)
    assert rows.shape == (0, 16) and plan.offs.tolist() == [0] * 6
    assert flag_gems.moe_unpermute(rows, plan).shape == (0, 16)
    assert torch.autograd.grad(rows.sum(), x)[0].shape == (0, 16)
    x = torch.ones(5, 0, device="cuda", requires_grad=True)
    ids = torch.ones(5, 2, dtype=torch.int32, device="cuda")
    rows, _, plan = flag_gems.moe_permute(x, ids, 6)
    w = torch.ones(5, 2, device="cuda", requires_grad=True)
    out = flag_gems.moe_unpermute(rows, plan, w)
    assert out.shape == (5, 0) and not torch.autograd.grad(out.sum(), w)[0].any()
    x = torch.ones(5, 16, device="cuda")
    rows, _, plan = flag_gems.moe_permute(x, ids[:, :0], 6)
    assert rows.shape == (0, 16) and plan.offs.tolist() == [0] * 6
    assert not flag_gems.moe_unpermute(rows, plan).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8])
def test_strides_and_alignment(dtype):
    g = _gen(1)
    t, k, e, h = 50, 3, 7, 96
    wide = (torch.randn(t, 256, device="cuda", generator=g) * 9).to(dtype)
    ids = _ids(t, e, k, g)
    want = _plan(ids, e)
    views = [wide[:, :h], wide[:, 16:16 + h], wide[:, 3:3 + h], wide[:, 1:1 + 95], wide[::1, ::2][:, :h],
             wide[:1, :h].expand(t, h), wide[:h, :t].t() if t <= 256 and h <= t else wide[:, :h].t().contiguous().t()]
    for x in views:
        for i in (ids, ids.t().contiguous().t(), torch.cat([ids, ids], 1)[:, :k]):
            rows, _, plan = flag_gems.moe_permute(x, i, e)
            _same_plan(plan, want)
            _check_permuted(x, rows, plan, k)
    if dtype == torch.int8:
        return
    plan = flag_gems.MoEPermutation(*want)
    big = torch.randn(t * k, 256, device="cuda", generator=g).to(dtype)
    w_wide = torch.randn(t, 9, device="cuda", generator=g)
    for y in (big[:, :h], big[:, 8:8 + h], big[:, 5:5 + h], big[:, ::2][:, :h], big[:1, :h].expand(t * k, h)):
        for w in (w_wide[:, 2:2 + k], w_wide[:, :k].t().contiguous().t(), w_wide[:, ::3], w_wide[:, :1].expand(t, k)):
            y_, w_ = y.detach().requires_grad_(), w.detach().requires_grad_()
            out = flag_gems.moe_unpermute(y_, plan, w_)
            _check_sum(out.detach(), y, plan.row_of_slot, w)
            d = torch.randn(t, 2 * h, device="cuda", generator=g).to(dtype)
            for d_out in (d[:, :h], d[:, 1:1 + h], d[:1, :1].expand(t, h)):
                got = torch.autograd.grad(out, (y_, w_), d_out, retain_graph=True)
                same = torch.autograd.grad(flag_gems.moe_unpermute(y_, plan, w_), (y_, w_), d_out.contiguous())
                assert torch.equal(got[0], same[0])
                torch.testing.assert_close(got[1], same[1], rtol=0, atol=2 * h * F32 * float(y.float().abs().max() * d.float().abs().max() * h))


def test_broadcast_inputs_and_leaves():
    """Gradients through .backward(), of an input that is broadcast and of weights used twice."""
    g = _gen(5)
    t, k, e, h = 20, 2, 4, 32
    ids = _ids(t, e, k, g)
    x = torch.randn(1, h, device="cuda", generator=g, requires_grad=True)
    w = torch.rand(t, k, device="cuda", generator=g, requires_grad=True)
    rows, _, plan = flag_gems.moe_permute(x.expand(t, h), ids, e)
    (flag_gems.moe_unpermute(rows, plan, w) + flag_gems.moe_unpermute(rows * 2, plan, w)).sum().backward()
    # out = 3 * sum_k w * x: its gradient is 3 * sum(w) for every value of x, 3 * sum(x) for every weight
    assert float((x.grad.double() - 3 * w.detach().double().sum()).abs().max()) <= float(w.detach().sum()) * 3 * 100 * F32
    mass = float(x.detach().abs().sum())
    assert float((w.grad.double() - 3 * x.detach().double().sum()).abs().max()) <= mass * 3 * 2 * h * F32
    with pytest.raises(RuntimeError, match="once_differentiable"):
        rows, _, plan = flag_gems.moe_permute(x.expand(t, h), ids, e)
        d, = torch.autograd.grad(rows.square().sum(), x, create_graph=True)
        d.sum().backward()


def test_no_gradient_without_asking():
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        rows, _, plan = flag_gems.moe_permute(x, ids, 2)
        out = flag_gems.moe_unpermute(x.repeat(2, 1), plan)
    assert not rows.requires_grad and not out.requires_grad
    rows, _, plan = flag_gems.moe_permute(x, ids, 2)
    assert rows.requires_grad and not any(p.requires_grad for p in plan)


class _Off:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.parametrize("native", [True, False])
def test_forward_mode_is_refused(native, monkeypatch):
    """Tangents of the inputs, and of a gradient on its way back, are not dropped."""
    if not native:
        monkeypatch.setattr(_cabi, "host", _Off())
    g = _gen(3)
    t, k, e, h = 6, 2, 4, 16
    ids, x, w = _ids(t, e, k, g), torch.randn(t, h, device="cuda", generator=g), torch.rand(t, k, device="cuda", generator=g)
    rows, _, plan = flag_gems.moe_permute(x, ids, e)
    out = flag_gems.moe_unpermute(rows, plan, w)
    with forward_ad.dual_level():
        def dual(v):
            return forward_ad.make_dual(v, torch.ones_like(v))

        for call in (lambda: flag_gems.moe_permute(dual(x), ids, e), lambda: flag_gems.moe_permute(dual(x.clone().requires_grad_()), ids, e),
                     lambda: flag_gems.moe_permute(x, ids, e, scale=dual(w)), lambda: flag_gems.moe_unpermute(dual(rows), plan, w),
                     lambda: flag_gems.moe_unpermute(rows, plan, dual(w)), lambda: flag_gems.moe_unpermute(dual(rows), plan)):
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call()
        x_, y_, w_ = (v.clone().requires_grad_() for v in (x, rows, w))
        for result in (flag_gems.moe_permute(x_, ids, e)[0], flag_gems.moe_unpermute(y_, plan, w_), flag_gems.moe_unpermute(y_, plan)):
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                (result * dual(torch.ones_like(result))).sum().backward()
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(flag_gems.moe_unpermute(dual(rows), plan, w), out)
    assert torch.equal(flag_gems.moe_unpermute(rows, plan, w), out)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_gradients_of_8_bit_floats_are_refused(dtype):
    g = _gen(4)
    ids, x = _ids(6, 4, 2, g), torch.randn(6, 16, device="cuda", generator=g).to(dtype)
    with pytest.raises(NotImplementedError, match="have no gradient"):
        flag_gems.moe_permute(x.clone().requires_grad_(), ids, 4)
    with torch.no_grad():
        rows, _, plan = flag_gems.moe_permute(x.clone().requires_grad_(), ids, 4)
    _check_permuted(x, rows, plan, 2)


@pytest.mark.parametrize("native", [True, False])
def test_rows_too_long_are_refused_alike(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_cabi, "host", _Off())
    x, ids = torch.empty(1, 1 << 31, dtype=torch.int8, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(NotImplementedError, match="size too large"):
        flag_gems.moe_permute(x, ids, 1)


def test_inf_and_nan_are_carried():
    x = torch.tensor([[1.0, float("inf")], [float("nan"), -0.0], [3.0, 65504.0]], device="cuda")
    ids = torch.tensor([[1, 0], [0, -1], [1, 1]], dtype=torch.int32, device="cuda")
    rows, _, plan = flag_gems.moe_permute(x, ids, 2)
    assert plan.row_of_slot.tolist() == [[2, 0], [1, ~5], [3, 4]]
    assert torch.equal(_bytes(rows), _bytes(torch.cat([x[[0, 1, 0, 2, 2]], torch.zeros(1, 2, device="cuda")])))
    out = flag_gems.moe_unpermute(rows, plan, torch.tensor([[0.0, 0.0], [1.0, float("nan")], [1.0, 1.0]], device="cuda"))
    assert out[0, 0] == 0 and out[0, 1].isnan() and out[1, 0].isnan() and out[1, 1] == 0 and out[2].tolist() == [6.0, 131008.0]


def test_results_do_not_depend_on_the_run():
    g = _gen(9)
    t, k, e, h = 4096, 8, 256, 256
    x = torch.randn(t, h, device="cuda", generator=g).bfloat16().requires_grad_()
    w = torch.rand(t, k, device="cuda", generator=g, requires_grad=True)
    ids = _ids(t, e, k, g)
    first = None
    for _ in range(3):
        rows, _, plan = flag_gems.moe_permute(x, ids, e)
        out = flag_gems.moe_unpermute(rows, plan, w)
        now = [rows.detach(), *plan, out.detach(), *torch.autograd.grad(out.float().square().sum(), (x, w))]
        first = first or now
        for a, b in zip(first, now):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """2.3e9 values, 4.6 GB of rows."""
    t, k, e, h = 40000, 8, 256, 7168
    g = _gen(2)
    x = torch.randn(t, h, device="cuda", generator=g).bfloat16().requires_grad_()
    w = torch.rand(t, k, device="cuda", generator=g, requires_grad=True)
    ids = _ids(t, e, k, g)
    rows, _, plan = flag_gems.moe_permute(x, ids, e)
    src = (plan.slot_of_row // k).long()
    for b in range(0, t * k, 40000):
        assert torch.equal(rows[b:b + 40000], x[src[b:b + 40000]])
    out = flag_gems.moe_unpermute(rows, plan, w)
    d_out = torch.randn(t, h, device="cuda", generator=g).bfloat16()
    d_rows, d_w = torch.autograd.grad(out, (rows, w), d_out, retain_graph=True)
    d_x, = torch.autograd.grad(rows, x, d_rows)
    last = slice(t - 500, t)
    pos = plan.row_of_slot[last]
    rr = rows.detach()
    _check_sum(out.detach()[last], rr, pos, w.detach()[last])
    _check_sum(d_x[last], d_rows, pos, None)
    want = d_out[last].double()[:, None, :] * w.detach()[last].double()[:, :, None]
    assert bool(((d_rows[pos.long()].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2 * F32)).all())
    prod = rr[pos.long()].double() * d_out[last].double()[:, None, :]
    assert bool(((d_w[last].double() - prod.sum(2)).abs() <= prod.abs().sum(2) * (h + 1) * F32 + prod.sum(2).abs() * F32).all())


def test_another_stream_two_at_once_and_graph_capture():
    g = _gen(4)
    t, k, e, h = 700, 8, 64, 512
    x = torch.randn(t, h, device="cuda", generator=g).bfloat16()
    w = torch.rand(t, k, device="cuda", generator=g)
    ids = _ids(t, e, k, g)
    ids2 = _ids(t, e, k, g)

    def both(i):
        rows, _, plan = flag_gems.moe_permute(x, i, e)
        return [rows, *plan, flag_gems.moe_unpermute(rows, plan, w)]

    want, want2 = both(ids), both(ids2)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(one):
            a = both(ids)
        with torch.cuda.stream(two):
            b = both(ids2)
        torch.cuda.synchronize()
        for p, q in zip(a + b, want + want2):
            assert torch.equal(p, q)

    d_out = torch.randn(t, h, device="cuda", generator=g).bfloat16()

    def step():
        x_, w_ = x.detach().requires_grad_(), w.detach().requires_grad_()
        rows, _, plan = flag_gems.moe_permute(x_, ids, e)
        out = flag_gems.moe_unpermute(rows * 2, plan, w_)
        return [out.detach(), *plan, *torch.autograd.grad(out, (x_, w_), d_out)]

    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    x.copy_(x.roll(3, 0))
    ids.copy_(ids2)
    w.mul_(0.5)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        for p, q in zip(out, step()):
            assert torch.equal(p, q)


def test_an_int8_expert_layer_of_its_parts():
    """Router ids -> sorted tokens -> int8 experts -> tokens, every step against the definition on what the step before gave."""
    g = _gen(6)
    t, k, e, h, inter = 301, 4, 16, 512, 256
    x = torch.randn(t, h, device="cuda", generator=g).bfloat16()
    logits = torch.randn(t, e, device="cuda", generator=g)
    w, ids = torch.empty(t, k, device="cuda"), torch.empty(t, k, dtype=torch.int32, device="cuda")
    flag_gems.topk_softmax(w, ids, torch.empty_like(ids), logits, True)
    w1, s1 = flag_gems.per_token_quant_int8(torch.randn(e, 2 * inter, h, device="cuda", generator=g) * 0.05)
    w2, s2 = flag_gems.per_token_quant_int8(torch.randn(e, h, inter, device="cuda", generator=g) * 0.05)
    s1, s2 = s1.view(e, 2 * inter), s2.view(e, h)

    def product(a, a_s, b, b_s, offs):
        out, begin = [], 0
        for i, end in enumerate(offs.tolist()):
            out.append((a[begin:end].double() @ b[i].double().t()) * a_s[begin:end].double() * b_s[i].double())
            begin = end
        return torch.cat(out)

    q, q_s = flag_gems.per_token_quant_int8(x)
    rows, row_s, plan = flag_gems.moe_permute(q, ids, e, scale=q_s)
    _same_plan(plan, _plan(ids, e))
    up = flag_gems.w8a8_int8_grouped_mm(rows, w1, row_s, s1, plan.offs)
    want = product(rows, row_s, w1, s1, plan.offs)
    assert bool(((up.double() - want).abs() <= want.abs() * (2.0 ** -8 + 4 * F32)).all())
    act = flag_gems.silu_and_mul(up[:, :inter], up[:, inter:])
    q2, q2_s = flag_gems.per_token_quant_int8(act)
    down = flag_gems.w8a8_int8_grouped_mm(q2, w2, q2_s, s2, plan.offs)
    want = product(q2, q2_s, w2, s2, plan.offs)
    assert bool(((down.double() - want).abs() <= want.abs() * (2.0 ** -8 + 4 * F32)).all())
    out = flag_gems.moe_unpermute(down, plan, w)
    _check_sum(out, down, plan.row_of_slot, w)
    # the shared expert of the same layer
    up = flag_gems.w8a8_int8_matmul(q, w1[0], q_s, s1[0])
    want = (q.double() @ w1[0].double().t()) * q_s.double() * s1[0].double()
    assert bool(((up.double() - want).abs() <= want.abs() * (2.0 ** -8 + 4 * F32)).all())
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t", [9, 3000])
def test_ids_and_maps_beyond_32_bits(ids_dtype, t):
    g = _gen(t)
    e, k, h = 6, 4, 40
    x = torch.randn(t, h, device="cuda", generator=g)
    ids = torch.randint(0, 12, (t, k), device="cuda", generator=g).to(ids_dtype)
    if ids_dtype == torch.int64:
        ids[::3, 0] += 2 ** 32  # no id of the map
        ids[1::3, 1] -= 2 ** 33
    else:
        ids[::3, 0] = torch.iinfo(torch.int32).max
        ids[1::3, 1] = torch.iinfo(torch.int32).min
    expert_map = torch.tensor([5, 0, 2 ** 32, -1, 2 ** 32 + 3, 1, 2, -2 ** 32, 3, 4, 2 ** 40 - 1, 6], device="cuda")
    rows, _, plan = flag_gems.moe_permute(x, ids, e, expert_map=expert_map)
    _same_plan(plan, _plan(ids, e, expert_map))
    _check_permuted(x, rows, plan, k)


def test_inference_mode():
    g = _gen(5)
    x, w = torch.randn(20, 64, device="cuda", generator=g).bfloat16(), torch.rand(20, 2, device="cuda", generator=g)
    ids = _ids(20, 8, 2, g)
    rows, _, plan = flag_gems.moe_permute(x, ids, 8)
    want = flag_gems.moe_unpermute(rows, plan, w)
    with torch.inference_mode():
        rows2, _, plan2 = flag_gems.moe_permute(x, ids, 8)
        assert torch.equal(flag_gems.moe_unpermute(rows2, plan2, w), want)
        plan2.row_of_slot.add_(0)  # an ordinary tensor in there
        assert rows2.is_inference() and plan2.row_of_slot.is_inference() and plan2.offs.is_inference()
    _same_plan([t.clone() for t in plan2], plan)


@pytest.mark.parametrize("h", [8, 36, 38, 39, 200, 2040])
@pytest.mark.parametrize("t,k,e", [(6, 3, 4), (300, 8, 64), (2501, 2, 9), (4800, 5, 320)])
def test_int8_rows_of_any_alignment(t, k, e, h):
    g = _gen(t + h)
    ids = _ids(t, e, k, g)
    ids[1] = e  # nowhere
    wide = torch.randint(-128, 128, (t, 2064), device="cuda", generator=g, dtype=torch.int8)
    scale = torch.rand(t, 3, device="cuda", generator=g)
    want = _plan(ids, e)
    for off in (0, 8, 4, 2, 1):
        x = wide[:, off:off + h]
        rows, row_scale, plan = flag_gems.moe_permute(x, ids, e, scale=scale)
        _same_plan(plan, want)
        _check_permuted(x, rows, plan, k)
        valid = int(plan.offs[-1])
        assert torch.equal(row_scale[:valid], scale[(plan.slot_of_row // k).long()][:valid]) and bool((row_scale[valid:] == 1.0).all())


@pytest.mark.parametrize("t,k,e,h", [(2000, 40, 64, 8), (1185, 3, 5, 128), (4737, 2, 8, 100), (5000, 1, 16, 1024), (2400, 6, 64, 264), (9473, 1, 2, 72)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_many_narrow_rows(t, k, e, h, dtype):
    test_permute(t, k, e, h, dtype)
    test_unpermute(t, k, e, h, dtype)
    test_gradients(t, k, e, h, dtype, torch.float32)
