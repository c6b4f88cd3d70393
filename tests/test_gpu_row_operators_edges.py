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


# ------------------------------------------------------------------------------------------------ AdamW
def test_adamw_refuses_a_state_that_was_replaced(cuda):
    """The step writes where the plan's state was when it was made: another tensor in one of its lists, another list, or other
    memory behind a tensor is refused; copying into the state is what loads another one."""
    for bits in (32, 8):
        params, grads = [rand(700, (300,), torch.bfloat16), rand(701, (70,), torch.bfloat16)], [rand(702, (300,), torch.bfloat16), rand(703, (70,), torch.bfloat16)]
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
