"""The row operators where values, states and places are far from ordinary: finite masks and large maxima, long runs of
8-bit states, decay below a parameter's step, device counters, updates that autograd has to see, gradients of slices.

Tolerances are those of test_gpu_row_operators.py, counted in roundings."""
import math

import pytest
import torch

from pixienn_b200 import ops

from test_gpu_row_operators import U, check_probs, gen, half_step, probs64, rand, within

pytestmark = pytest.mark.gpu

INF = float("inf")


# ------------------------------------------------------------------------------------------------ finite masks
def masked_rows(dtype, v, values):
    """Rows with none, half, 95 %, a contiguous part, all but three, all but one and all of their classes at each of `values`,
    and rows whose largest value is far from zero."""
    keep = torch.rand(v, device="cuda", generator=gen(601))
    at = torch.arange(v, device="cuda")
    gone = [keep < 0.5, keep < 0.95, at < 3 * v // 4, at >= v // 4, (at != 5) & (at != v // 2) & (at != v - 1), at != v - 2, at >= 0]
    rows = [rand(602, (1, v), dtype, 2.5)[0]]
    for k, value in enumerate(values):
        for mask in gone:
            rows.append(rand(603 + k, (1, v), dtype, 2.5)[0].masked_fill(mask, value))
    for value in values:                                  # the mask's value is the row's largest but for its neighbours
        rows.append((value * (1 + rand(620, (1, v)).abs()[0])).to(dtype))
        rows.append((-value * (1 - rand(621, (1, v)).abs()[0] / 16)).to(dtype))
    rows.append(rand(622, (1, v), dtype, 2.5)[0].masked_fill(gone[2], values[0]).masked_fill(gone[0], -INF))
    return torch.stack(rows)


MASKS = {torch.float32: (-1e4, -1e7, -1e9, -1e10, -1e20, -1e30), torch.bfloat16: (-1e4, -1e7, -1e9, -1e10, -1e20, -1e30),
         torch.float16: (-1e3, -1e4, -6e4)}


def check_gradient(x, target, r, lp, h, temperature):
    """log_probs_backward against the formula, as the other gradient tests count it."""
    n, v = x.shape
    g, gh = rand(630, (n,)), rand(631, (n,))
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    hot = torch.zeros_like(p).scatter_(1, target[:, None], 1.0)
    gd, hd = g.double()[:, None], gh.double()[:, None]
    want = (gd * (hot - p) - hd * p * (lp0 + h[:, None])) / temperature
    size = (gd.abs() * (hot + p) + hd.abs() * p * (lp0.abs() + h[:, None].abs() + math.log(v + 1) + 1)) / temperature
    tol = size * U * ((v / 512 + 40) + 200)
    # 2^d below 2^-126 is flushed to 0: what is lost is p <= 2^-126 times (|g| + |gH| (entropy + |ln p|)) / T, |ln p| up to
    # the 103 at which fp32 itself has nothing left
    lost = 2.0 ** -126 * (gd.abs() + hd.abs() * (h[:, None].abs() + 103)) / temperature
    got = ops.log_probs_backward(x, target, r.stats, g, dentropy=gh, temperature=temperature)
    within(got, want, tol + half_step(x.dtype, want.abs() + tol) + lost)


@pytest.mark.parametrize("dtype", list(MASKS))
@pytest.mark.parametrize("v", [1030, 2100, 9001, 50003, 131072])
@pytest.mark.parametrize("temperature", [1.0, 0.75, 0.125, 2.0 ** -20])
def test_log_probs_with_finite_masks(cuda, dtype, v, temperature):
    """(The temperatures are fp32 numbers, so that both sides divide by the same.)"""
    x = masked_rows(dtype, v, MASKS[dtype])
    n = len(x)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen(640))
    target[::2] = x[::2].argmax(1)
    for top in (0, 1, 20):
        r, lp = check_probs(x, target, temperature, top)
    (_, h, _, _), _ = probs64(x, target, temperature, 0)
    check_gradient(x, target, r, lp, h, temperature)
    for k in (3, 15, n - 2):                              # a row by itself, which more blocks share
        check_probs(x[k:k + 1], target[k:k + 1], temperature, 3)
        check_probs(x[k:k + 1], target[k:k + 1], temperature)


@pytest.mark.parametrize("dtype", list(MASKS))
@pytest.mark.parametrize("v", [4100, 12000])
def test_log_probs_of_many_rows_with_finite_masks(cuda, dtype, v):
    """Enough rows for the forms with few threads to a row."""
    rows = masked_rows(dtype, v, MASKS[dtype])
    x = rows.repeat(-(-1200 // len(rows)), 1)
    target = torch.randint(0, v, (len(x),), device="cuda", generator=gen(641))
    for temperature, top in ((1.0, 0), (0.125, 0), (1.0, 2), (0.125, 2)):
        got = ops.log_probs(x, target, top=top, temperature=temperature)
        few, _ = check_probs(rows, target[:len(rows)], temperature, top)
        assert not bool(got.entropy.isnan().any()) and not bool(got.logp.isnan().any())
        tol = 2 * U * ((8 * v / 512 + 40) + 150) * (1 + math.log(v + 1) + few.entropy.double().abs())
        within(got.entropy[:len(rows)], few.entropy, tol)
        within(got.logp[:len(rows)], few.logp, tol + 12 * U * few.logp.double().abs().nan_to_num(posinf=0.0))
        for k in range(len(rows), len(x), len(rows)):      # the same rows again, at other distances from a boundary
            m = min(len(rows), len(x) - k)
            within(got.entropy[k:k + m], few.entropy[:m], tol[:m])
            assert top == 0 or torch.equal(got.top_index[k:k + m], few.top_index[:m])


@pytest.mark.parametrize("v", [1030, 2100, 9001, 70000])
@pytest.mark.parametrize("temperature", [1.0, 0.125])
def test_log_probs_around_the_limits_of_the_origin(cuda, v, temperature):
    """Rows whose values lie on both sides of -2^24 and 2^24, and of twice that, in units of temperature / log2(e): none of their
    terms may be lost, on whichever side a thread's, a block's or the row's maximum lies."""
    edge = 2.0 ** 24 * temperature * math.log(2.0)
    spread = rand(650, (1, v))[0] * 3 * temperature
    rows = []
    for at in (-edge, edge, -2 * edge, 2 * edge):
        for off in (-12, -6, -3, 0, 3, 6, 12):
            rows.append(at + off * temperature + spread)
        rows.append((at + spread).sort().values)
        rows.append((at + spread).sort(descending=True).values)
    x = torch.stack(rows)
    target = x.argmax(1)
    target[1::3] = v // 2
    for top in (0, 4):
        r, lp = check_probs(x, target, temperature, top)
    (_, h, _, _), _ = probs64(x, target, temperature, 0)
    check_gradient(x, target, r, lp, h, temperature)
    many = x.repeat(40, 1)
    check_probs(many, target.repeat(40), temperature)
    for k in (0, 3, 7, 8, 12):
        check_probs(x[k:k + 1], target[k:k + 1], temperature, 4)


# ------------------------------------------------------------------------------------------------ AdamW
def test_adamw_refuses_a_state_that_was_replaced(cuda):
    """The step writes where the plan's state was when it was made: another tensor in one of its lists, another list, or other
    memory behind a tensor is refused; copying into the state is what loads another one."""
    for bits in (32, 8):
        params, grads = ([rand(seed + k, (n,), torch.bfloat16) for k, n in enumerate((300, 70))] for seed in (700, 702))
        plan = ops.AdamW(params, state_bits=bits, master=True)
        names = ["m", "v", "master"] + (["m_scale", "v_scale"] if bits == 8 else [])
        old = {name: list(getattr(plan, name)) for name in names}              # (kept, so that nothing is freed)
        before = [p.clone() for p in params]
        for name in names:
            getattr(plan, name)[1] = old[name][1].clone()
            with pytest.raises(RuntimeError, match=name):
                plan.step(grads, rate=1e-2, t=1)
            getattr(plan, name)[1] = old[name][1]
            setattr(plan, name, [t.clone() for t in old[name]])
            with pytest.raises(RuntimeError, match=name):
                plan.step(grads, rate=1e-2, t=1)
            setattr(plan, name, old[name][:1])
            with pytest.raises(RuntimeError, match=name):
                plan.step(grads, rate=1e-2, t=1)
            setattr(plan, name, list(old[name]))
            memory = old[name][0].data
            old[name][0].data = memory.clone()
            with pytest.raises(RuntimeError, match=name):
                plan.step(grads, rate=1e-2, t=1)
            old[name][0].data = memory
        assert all(torch.equal(p, b) for p, b in zip(params, before))
        plan.step(grads, rate=1e-2, t=1)
        assert not torch.equal(params[0], before[0])
        plan.m[0].copy_(torch.zeros_like(plan.m[0].float()))
        plan.step(grads, rate=1e-2, t=2)


def test_adamw_counter_below_one_leaves_everything(cuda):
    """t counts from 1; a device counter that is not there yet (a step replayed before it is raised) changes nothing, where
    1 - beta^0 = 0 would divide."""
    for bits in (32, 8):
        params, grads = [rand(710, (300,)), rand(711, (5,))], [rand(712, (300,)), rand(713, (5,))]
        plan = ops.AdamW(params, state_bits=bits)
        plan.step(grads, rate=1e-2, t=1)
        held = params + plan.m + plan.v + (plan.m_scale + plan.v_scale if bits == 8 else [])
        before = [x.clone() for x in held]
        for t in (0, -1, -(1 << 40)):
            plan.step(grads, rate=1e-2, t=torch.tensor([t], device="cuda"))
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(held, before))
        plan.step(grads, rate=1e-2, t=torch.tensor([2], device="cuda"))
        assert not torch.equal(params[0], before[0]) and bool(params[0].isfinite().all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("rate,decay", [(1e-4, 0.01), (3e-6, 0.1), (1e-3, 0.05)])
def test_adamw_decay_of_few_units_is_not_quantised(cuda, bits, rate, decay):
    """With nothing but decay (gradient and moments 0) the parameter is p - rate decay p, rounded once: off by half of its own
    step, and U of the decay itself for each of its two products, whatever rate * decay is next to 2^-24."""
    p = rand(720, (20000,))
    plan, before = ops.AdamW([p], state_bits=bits), p.double()
    plan.step([torch.zeros_like(p)], rate=rate, t=1, weight_decay=decay)
    shrink = float(torch.tensor(rate, dtype=torch.float32).double() * torch.tensor(decay, dtype=torch.float32).double())
    want = before * (1 - shrink)
    step = (torch.nextafter(p.abs(), torch.full_like(p, INF)) - p.abs()).double()
    within(p, want, step / 2 + 2 * U * shrink * before.abs())


def decoded(codes, scale):
    return codes.double() * scale.double().repeat_interleave(256)[:codes.numel()]


@pytest.mark.parametrize("dtype,gtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                         (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_seeded_codes_are_neighbours_and_fair(cuda, dtype, gtype, master, shift):
    """With a seed each code is the value's neighbour above or below, and their mean error is none: that of n values is within
    five times 1/2 step / sqrt(n) (a code's error has a deviation of at most half a step), and 2^-17 of a step for 16 random
    bits.  Everything else is as without a seed."""
    if master and dtype == torch.float32:
        return
    sizes = [200003, 77, 512]
    made = lambda s: [rand(s + k, (n + shift,), dtype, 0.05)[shift:] for k, n in enumerate(sizes)]  # noqa: E731
    grads = [[rand(s + k, (n + shift,), gtype, 0.01)[shift:] for k, n in enumerate(sizes)] for s in (740, 750)]
    a, b = made(730), made(730)
    pa, pb = ops.AdamW(a, state_bits=8, master=master, seed=5), ops.AdamW(b, state_bits=8, master=master)
    pa.step(grads[0], rate=1e-2, t=1)
    pb.step(grads[0], rate=1e-2, t=1)
    assert all(torch.equal(x, y) for x, y in zip(a + pa.m_scale + pa.v_scale, b + pb.m_scale + pb.v_scale))
    b1, b2 = (float(torch.tensor(x, dtype=torch.float32)) for x in (0.9, 0.999))
    m0, r0 = ([decoded(q, s) for q, s in zip(*z)] for z in ((pa.m, pa.m_scale), (pa.v, pa.v_scale)))
    pa.step(grads[1], rate=1e-2, t=2)
    errors = []
    for k, n in enumerate(sizes):
        g = grads[1][k].double()
        for q, s, want in ((pa.m[k], pa.m_scale[k], b1 * m0[k] + (1 - b1) * g),
                           (pa.v[k], pa.v_scale[k], (b2 * r0[k].square() + (1 - b2) * g * g).sqrt())):
            each = s.double().repeat_interleave(256)[:n]
            at = (want / each).abs()
            step = torch.exp2(torch.floor(torch.log2(at.clamp(min=2.0 ** -6))) - 3)          # between codes around the value
            # a neighbour: less than a step away, 16 U of the value for what is computed on the way, which can lie over a
            # code's value itself (an error of a whole step of the next octave: twice as long)
            off = (decoded(q, s) - want) / each
            floor = (q is pa.v[k]) & (at < 2.0 ** -9)                                        # kept at the smallest code
            assert bool((off.abs() <= torch.where(floor, 2.0 ** -9, step) + 2 * step * (at * 16 * U > step * 2.0 ** -17) + at * 16 * U).all())
            if n > 100000:
                errors.append((off / step * want.sign())[(at > 2.0 ** -6) & (at < 448 * 0.999)])
        assert bool(((pa.v[k].float() > 0) == (r0[k].square() + g * g > 0)).all())
    for e in errors:
        assert abs(float(e.mean())) <= 2.5 / math.sqrt(e.numel()) + 2.0 ** -17 + 1e-4
        assert 0.1 < float(e.abs().mean()) < 0.5              # (to nearest it is at most 0.25; at random the mean of 2 f (1 - f) is 1/3)


def test_adamw_seeded_steps_repeat_and_differ(cuda):
    """The same bits for the same seed, t and places, whatever the alignment and however t is given; others for another seed,
    t or tensor."""
    n = 5000
    def state(seed, t, device_t=False, shift=0, count=2):
        params = [rand(760, (n + shift,))[shift:].clone() if not shift else rand(760, (n,)).clone() for _ in range(count)]
        if shift:
            params = [torch.empty(n + shift, device="cuda")[shift:].copy_(p) for p in params]
        plan = ops.AdamW(params, state_bits=8, seed=seed)
        grads = [rand(761, (n,), scale=0.01) for _ in range(count)]
        plan.step(grads, rate=1e-3, t=torch.tensor([t], device="cuda") if device_t else t)
        return [x.float() for x in plan.m + plan.v]
    one = state(7, 3)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    assert same(one, state(7, 3)) and same(one, state(7, 3, device_t=True)) and same(one, state(7, 3, shift=1))
    many = state(7, 3, count=450)                             # more than one launch
    assert same(one[:2], many[:2]) and same(one[2:], many[450:452])
    assert not torch.equal(many[0], many[1]) and not torch.equal(many[399], many[400]) and not torch.equal(many[0], many[400])
    for other in (state(8, 3), state(7 + (1 << 32), 3), state(7, 4), state(7, 3 + (1 << 32))):
        assert 0.05 < float((other[0] != one[0]).float().mean()) < 0.95
    for bad in (0, -1, 1 << 64):
        with pytest.raises(ValueError):
            ops.AdamW([torch.zeros(4, device="cuda")], state_bits=8, seed=bad)
    with pytest.raises(ValueError):
        ops.AdamW([torch.zeros(4, device="cuda")], seed=1)


def test_adamw_seeded_state_keeps_what_is_not_finite_and_zero(cuda):
    """A gradient of 0 on a fresh state leaves zeros; one that is not finite spoils its block and no other, as without a seed."""
    p = [rand(770, (1024,))]
    plan = ops.AdamW(p, state_bits=8, seed=3)
    plan.step([torch.zeros(1024, device="cuda")], rate=1e-3, t=1)
    assert bool((plan.m[0].float() == 0).all()) and bool((plan.v[0].float() == 0).all())
    for bad in (float("nan"), INF, -INF):
        q = [p[0].clone()]
        plan, plain = ops.AdamW(q, state_bits=8, seed=3), ops.AdamW([p[0].clone()], state_bits=8)
        g = rand(771, (1024,))
        g[300] = bad
        plan.step([g], rate=1e-3, t=1)
        plain.step([g], rate=1e-3, t=1)
        for x, y in ((plan.m[0], plain.m[0]), (plan.v[0], plain.v[0])):
            assert torch.equal(x.float().isnan(), y.float().isnan()) and not bool(x[:256].float().isnan().any() | x[512:].float().isnan().any())
        assert torch.equal(q[0].isnan(), plain.params[0].isnan())


def test_adamw_long_run_of_seeded_8_bit_state_follows_32_bits(cuda):
    """1300 steps of gradients whose sizes spread over orders of magnitude within a block; after 300 those of every other
    element fall to a tenth.  The root of v of 8-bit state over that of 32-bit state: a code's error is fair, so that the mean
    over many elements is off by half of the ratio's variance at most.  That variance: what rounding adds each step, |move| *
    code step, over twice the rate 1 - beta2 at which v forgets: a move of about (1 - beta2) / 2 of the root for what the
    gradient says and as much for the scale's own, codes 1/8 apart at most: 1/16 and a little more where gradients have fallen.
    So: mean within 8 %, 90 % of the elements within a factor of 2.  (To nearest the fallen half is 2.0 times too large
    after these 1000 steps and 6.8 after 4000, the other at 0.77 of what it should be.)"""
    n = 64 * 256
    size = torch.exp(rand(780, (n,))) * 0.01
    a, b = [torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")]
    small, wide = ops.AdamW(a, state_bits=8, seed=11), ops.AdamW(b)
    g = gen(781)
    for t in range(1, 1301):
        if t == 301:
            size[::2] *= 0.1
        grad = [torch.randn(n, device="cuda", generator=g) * size]
        small.step(grad, rate=1e-4, t=t)
        wide.step(grad, rate=1e-4, t=t)
        if t in (300, 800, 1300):
            ratio = decoded(small.v[0], small.v_scale[0]) / wide.v[0].double().sqrt()
            for part in (ratio[::2], ratio[1::2]):
                assert 0.92 <= float(part.mean()) <= 1.08
                assert float(torch.quantile(part, 0.05)) >= 0.5 and float(torch.quantile(part, 0.95)) <= 2.0
    # both have moved the parameters alike: the sum of 1300 updates of a rate each
    assert float((a[0] - b[0]).double().norm() / b[0].double().norm()) <= 0.25


# ------------------------------------------------------------------------------------------------ autograd sees what is written
def test_updates_in_place_are_seen_by_autograd(cuda):
    """A graph that saved a tensor which one of the calls then writes refuses its backward pass, as after any update in place;
    one whose tensors were read only goes through."""
    def saved(t):
        t = t.detach().requires_grad_(True)
        u = t * 1.0                                       # not a leaf, so that it may be written
        return u, (u * u).sum()

    def changed(call, *shape):
        u, loss = saved(rand(790, shape))
        call(u)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()

    w, x, target = rand(791, (32,)), rand(792, (6, 32)), torch.zeros(6, dtype=torch.int64, device="cuda")
    rstd = ops.rms_norm(x, w)[2]
    stats, d = ops.log_probs(x, target).stats, rand(793, (6,))
    changed(lambda u: ops.rms_norm(x, w, out=u), 6, 32)
    changed(lambda u: ops.rms_norm(x, w, residual=x, residual_out=u), 6, 32)
    changed(lambda u: ops.rms_norm(u, w, out=u), 6, 32)
    changed(lambda u: ops.rms_norm_backward(x, x, w, rstd, dx=u), 6, 32)
    changed(lambda u: ops.rms_norm_backward(x, x, w, rstd, dweight=u), 32)
    changed(lambda u: ops.log_probs_backward(x, target, stats, d, dx=u), 6, 32)
    for bits in (32, 8):
        changed(lambda u: ops.AdamW([u], state_bits=bits).step([x], rate=1e-2, t=1), 6, 32)
    q = torch.empty(6, 32, device="cuda", dtype=torch.float8_e4m3fn)
    before = q._version
    ops.rms_norm_e4m3(x, w, out=q)
    assert q._version > before
    u, loss = saved(x)
    for call in (lambda: ops.rms_norm(u, w, residual=u), lambda: ops.rms_norm_backward(u, u, w, rstd, dresidual=u),
                 lambda: ops.log_probs(u, target), lambda: ops.log_probs_backward(u, target, stats, d),
                 lambda: ops.AdamW([w.clone()]).step([u[0].detach()], rate=1e-2, t=1)):
        call()
    loss.backward()
    with torch.inference_mode():                          # tensors without a counter
        p = [torch.ones(8, device="cuda")]
        ops.AdamW(p).step([p[0].clone()], rate=1e-2, t=1)
        ops.rms_norm(p[0], out=p[0])


# ------------------------------------------------------------------------------------------------ gradients of slices
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_log_probs_gradient_of_a_slice_is_dense_and_aligned_like_it(cuda, dtype):
    """The gradient of a few rows of a large tensor takes the memory of a few rows; its rows lie at x's distances from a
    16-byte boundary, so that whole vectors are used; its values are those of the rows in a tensor of their own."""
    big = rand(800, (6, 40, 1003), dtype, 2.0)
    odd = rand(801, (6 * 1003 + 3,), dtype, 2.0)
    wide = rand(802, (3, 4, 5, 1100), dtype, 2.0)
    slices = [big[:, -1], big[:, 3:5], big[2], big[:, 7:8], big[1:2, :9], big[:, :, 5:900][:, 39], odd[3:].view(6, 1003), odd[1:1004],
              wide[..., 7:1010], wide[:, :, 2:3, :64], wide[1, :, 4], big[:, :0], big.view(240, 1003)[::40, 1:]]
    for x in slices:
        lead, v = x.shape[:-1], x.shape[-1]
        target = torch.randint(-1, v, lead, device="cuda", generator=gen(803))
        r, (d, dh) = ops.log_probs(x, target), (rand(k, (lead.numel(),)).view(lead) for k in (804, 805))
        dense = x.clone(memory_format=torch.contiguous_format)
        want = ops.log_probs_backward(dense, target, r.stats, d, dentropy=dh)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        got = ops.log_probs_backward(x, target, r.stats, d, dentropy=dh)
        used = torch.cuda.memory_allocated() - before
        rows = x.numel() // v
        assert used <= (rows * (v + 8) + len(x) * 8 + 8) * x.element_size() + 512
        assert got.shape == x.shape
        size = (d.abs() + dh.abs() * 20).double()[..., None]
        within(got, want, 8 * U * size + half_step(dtype, want.double()) * 2)    # (the two may add up a row's elements alike or not)
        if rows:
            mine, theirs = got.view(got.shape) if got.dim() > 1 else got[None], x if x.dim() > 1 else x[None]
            for index in torch.cartesian_prod(*[torch.arange(k) for k in theirs.shape[:-1]]).reshape(-1, theirs.dim() - 1)[:50]:
                at = tuple(int(k) for k in index)
                assert (mine[at].data_ptr() - theirs[at].data_ptr()) % 16 == 0


def test_log_probs_gradient_in_place_whatever_unused_strides_say(cuda):
    """The outer stride of a single group and the row stride of a single row say nothing: dx may be x, however they differ."""
    import ctypes as C
    from pixienn_b200 import capi
    x, target = rand(810, (4, 100)), torch.tensor([1, 2, -1, 99], device="cuda")
    r, d = ops.log_probs(x, target), rand(811, (4,))
    want = ops.log_probs_backward(x, target, r.stats, d)
    for rows, inner, outer, dx_outer, stride, dx_stride in ((4, 4, 400, 0, 100, 0), (4, 4, 7, 1 << 40, 100, 100), (1, 0, 0, 0, 100, 300), (1, 1, 5, 9, 200, 0)):
        mine = x[:rows].clone()
        desc = capi.LogProbsBackwardDesc(mine.data_ptr(), target.data_ptr(), r.stats.data_ptr(), d.data_ptr(), None, mine.data_ptr(), rows, inner,
                                         outer, stride, dx_outer, dx_stride, 100, capi.F32, 1, 1.0)
        capi.check(capi.lib().pxe_log_probs_backward(torch.cuda.current_stream().cuda_stream, C.byref(desc)))
        assert torch.equal(mine, want[:rows])
