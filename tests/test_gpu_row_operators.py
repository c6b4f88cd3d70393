"""The row operators (RMS norm with residual and 8-bit output, log probabilities with alternatives, AdamW over many
tensors) against plain forms in 64 bits, at the sizes, strides, masks and values where they can go wrong.

Tolerances count roundings: half a step of the output's type (finfo.eps / 2 of the value), U = 2^-24 for each operation
in 32 bits on the way, and for a sum of n terms U times the longest chain of additions that one term passes through
(the terms of one thread, then the tree)."""
import math

import pytest
import torch

from pixienn_b200 import capi, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = float("inf"), float("nan")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand(seed, shape, dtype=torch.float32, scale=1.0, pad=0, shift=0):
    """Normal values in a buffer `pad` columns wider, starting `shift` elements in."""
    n = 1
    for k in shape[:-1]:
        n *= k
    flat = torch.randn(n * (shape[-1] + pad) + shift, device="cuda", generator=gen(seed)).mul_(scale).to(dtype)
    return flat[shift:].view(*shape[:-1], shape[-1] + pad)[..., :shape[-1]]


def within(got, want, tol):
    """|got - want| <= tol everywhere, the same infinities (a value that got's type cannot hold is one) and NaNs."""
    want = torch.where(want.to(got.dtype).isinf(), want.to(got.dtype).double(), want.double())
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), "NaNs differ"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), "infinities differ"
    fine = ~(inf | want.isnan())
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"over the tolerance by {float(over.max()):.3g} of {float(torch.as_tensor(tol).max()):.3g}"


def half_step(dtype, value):
    """Rounding to dtype: half a step, or half the smallest subnormal."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


# ------------------------------------------------------------------------------------------------ norm
def norm_chain(c):
    """Longest chain of a row's sum: at most 64 terms of one thread (or a 1024th of the row), two trees of five."""
    return max(64, -(-c // 1024) + 8) + 10


def norm64(x, weight, residual, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.double()
    rstd = 1.0 / (f.square().mean(-1) + eps).sqrt()
    w = 1.0 if weight is None else weight.double()
    return h, rstd, f * rstd[..., None] * w


NORM_SHAPES = [(1, 1), (3, 7), (5, 32), (1, 4096), (2, 33), (300, 64), (4, 257), (7, 1023), (6, 1024), (3, 2048), (2, 5120), (2, 8191),
               (3, 16384), (2, 20002), (1, 65536), (149, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (1, 3), (2, 2)])
def test_rms_norm_equals_64_bits(cuda, dtype, shape, pad, shift):
    eps = 1e-5
    for with_res, wtype in ((True, torch.float32), (False, dtype), (True, None)):
        x = rand(1, shape, dtype, 1.5, pad, shift)
        res = rand(2, shape, dtype, 2.0, pad, shift) if with_res else None
        w = rand(3, (shape[-1],), wtype) if wtype is not None else None
        y, h, rstd = ops.rms_norm(x, w, residual=res, eps=eps)
        h64, r64, y64 = norm64(x, w, res, eps)
        assert torch.equal(h, h64) and (with_res or h is x)
        rel = (norm_chain(shape[-1]) / 2 + 6) * U
        within(rstd, r64, r64 * rel)
        within(y, y64, y64.abs() * (rel + 3 * U) + half_step(dtype, y64 * (1 + 1e-3)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 100), (1, 4096), (33, 128), (5, 1000), (3, 5120), (2, 8191), (1, 40000), (200, 320)])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1), (2, 2)])
def test_rms_norm_e4m3_equals_64_bits(cuda, dtype, shape, group, pad, shift):
    x = rand(4, shape, dtype, 1.0, pad, shift)
    res = rand(5, shape, dtype, 1.0, pad, shift)
    w = rand(6, (shape[-1],))
    x[0, :min(32, shape[-1])] = 0                        # a group of nothing
    res[0, :min(32, shape[-1])] = 0
    q, scale, h, rstd = ops.rms_norm_e4m3(x, w, residual=res, eps=1e-6, group=group)
    h64, r64, y64 = norm64(x, w, res, 1e-6)
    assert torch.equal(h, h64) and q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    n, c = shape
    g = group or c
    groups = -(-c // g)
    assert scale.shape == (n, groups)
    wide = torch.zeros(n, groups * g, dtype=torch.float64, device="cuda")
    wide[:, :c] = y64
    s64 = (wide.view(n, groups, g).abs().amax(-1) / 448).clamp(min=2.0 ** -126)
    rel = (norm_chain(c) / 2 + 9) * U
    within(scale, s64, s64 * (rel + 2 * U))
    each = s64.repeat_interleave(g, 1)[:, :c]
    got = q.double() * scale.double().repeat_interleave(g, 1)[:, :c]
    # half a step of the code (2^-4 of the value, 2^-10 of the scale among the smallest), after a value off by rel
    within(got, y64, y64.abs() * (2.0 ** -4 * 1.001 + 2 * rel) + each * 2.0 ** -10 * 1.001)


MANY = [(torch.bfloat16, 5000, 512), (torch.bfloat16, 2500, 2048), (torch.float16, 2600, 4096), (torch.bfloat16, 1300, 5120), (torch.float32, 1500, 4096),
        (torch.bfloat16, 700, 16384), (torch.float32, 10000, 256), (torch.float16, 1203, 8192), (torch.bfloat16, 3001, 1032)]


@pytest.mark.parametrize("dtype,n,c", MANY)
@pytest.mark.parametrize("pad", [0, 64])
def test_norms_of_many_rows_equal_64_bits(cuda, dtype, n, c, pad):
    """Enough rows for every block to take several, in whole vectors: forward in both outputs and backward, with and
    without the residual, in place as well."""
    w = rand(46, (c,))
    rel = (norm_chain(c) / 2 + 9) * U
    for with_res in (True, False):
        x = rand(47, (n, c), dtype, 1.0, pad)
        res = rand(48, (n, c), dtype, 1.0, pad) if with_res else None
        y, h, rstd = ops.rms_norm(x, w, residual=res, eps=1e-6)
        h64, r64, y64 = norm64(x, w, res, 1e-6)
        assert torch.equal(h, h64)
        within(rstd, r64, r64 * rel)
        within(y, y64, y64.abs() * rel + half_step(dtype, y64 * (1 + 1e-3)))
        for group in (0, 128):
            q, scale, h2, _ = ops.rms_norm_e4m3(x, w, residual=res, eps=1e-6, group=group)
            g = group or c
            groups = -(-c // g)
            wide = torch.zeros(n, groups * g, dtype=torch.float64, device="cuda")
            wide[:, :c] = y64
            s64 = (wide.view(n, groups, g).abs().amax(-1) / 448).clamp(min=2.0 ** -126)
            within(scale, s64, s64 * (rel + 2 * U))
            each = s64.repeat_interleave(g, 1)[:, :c]
            within(q.double() * scale.double().repeat_interleave(g, 1)[:, :c], y64, y64.abs() * (2.0 ** -4 * 1.001 + 2 * rel) + each * 2.0 ** -10 * 1.001)
            assert torch.equal(h2, h)
        dy, dres = rand(49, (n, c), dtype, 1.0, pad), rand(50, (n, c), dtype, 1.0, pad) if with_res else None
        dx, dw = ops.rms_norm_backward(dy, h, w, rstd, dresidual=dres)
        hd, u, r = h.double(), dy.double() * w.double(), rstd.double()[:, None]
        mean, terms = (u * hd).mean(1, keepdim=True), dy.double() * hd * r
        dx64 = r * (u - hd * r * r * mean) + (dres.double() if with_res else 0.0)
        spread = r * (u.abs() + hd.abs() * r * r * (u * hd).abs().mean(1, keepdim=True) * (norm_chain(c) + 8)) * 6 * U
        within(dx, dx64, spread + 2 * U * dx64.abs() + half_step(dtype, dx64.abs() + spread))
        within(dw, terms.sum(0), (n / 148 + 8 + 40 + 32 + 3) * U * terms.abs().sum(0))
        if with_res:
            xin, rin = x.clone(), res.clone()
            y2, h2, _ = ops.rms_norm(xin, w, residual=rin, eps=1e-6, out=xin, residual_out=rin)
            assert torch.equal(y2, y) and torch.equal(h2, h)
            again, dw2 = ops.rms_norm_backward(dy, h, w, rstd, dresidual=dres, dx=dres)
            assert torch.equal(again, dx) and torch.equal(dw2, dw)


def test_rms_norm_special_rows(cuda):
    """Zeros, NaN, infinities and values whose squares overflow stay in their row and mean what IEEE arithmetic says."""
    for dtype in TYPES:
        for c in (40, 1024, 70000):
            x = rand(7, (7, c), dtype)
            x[0] = 0
            x[1, c // 2] = NAN
            x[2, 3] = INF
            x[3] = torch.finfo(dtype).max
            x[4, c - 1] = -INF
            y, _, rstd = ops.rms_norm(x, None, eps=1e-6)
            f = x.float()
            ref_r = torch.rsqrt(f.square().mean(1) + 1e-6)
            ref = f * ref_r[:, None]
            if dtype != torch.float16:                   # 65504^2 * c stays finite in 32 bits
                assert float(rstd[3]) == 0 and bool((y[3] == 0).all())
            assert bool((y[0] == 0).all()) and bool(y[1].isnan().all())
            assert torch.equal(y[[1, 2, 4]].isnan(), ref[[1, 2, 4]].isnan()) and float(rstd[2]) == 0
            clean = ops.rms_norm(x[5:].contiguous(), None, eps=1e-6)[0]
            assert torch.equal(y[5:], clean)
            q, scale, _, _ = ops.rms_norm_e4m3(x, None, eps=1e-6, group=32)
            assert bool((q[0].float() == 0).all()) and float(scale[0, 0]) == 2.0 ** -126
            assert bool(scale[1].isnan().all()) and bool(q[1].float().isnan().all())
            assert not bool(q[5:].float().isnan().any())
            # eps = 0 on a row of zeros: 0 * inf
            assert bool(ops.rms_norm(x[:1], None, eps=0.0)[0].isnan().all())


def test_rms_norm_in_place_and_neighbours(cuda):
    """y on x, h on the residual, column slices of one buffer; what lies around them keeps its bits."""
    for dtype, c, pad in ((torch.bfloat16, 512, 24), (torch.float32, 1001, 3), (torch.float16, 70, 2), (torch.float32, 30001, 5)):
        x, res, w = rand(8, (9, c), dtype), rand(9, (9, c), dtype), rand(10, (c,))
        y0, h0, r0 = ops.rms_norm(x, w, residual=res)
        bx, br = rand(11, (9, c + pad), dtype), rand(12, (9, c + pad), dtype)
        keep_x, keep_r = bx.clone(), br.clone()
        bx[:, :c], br[:, :c] = x, res
        y, h, r = ops.rms_norm(bx[:, :c], w, residual=br[:, :c], out=bx[:, :c], residual_out=br[:, :c])
        assert torch.equal(bx[:, :c], y0) and torch.equal(br[:, :c], h0) and torch.equal(r, r0)
        assert torch.equal(bx[:, c:], keep_x[:, c:]) and torch.equal(br[:, c:], keep_r[:, c:])
        bx[:, :c], br[:, :c] = x, res                    # the other way round
        ops.rms_norm(bx[:, :c], w, residual=br[:, :c], out=br[:, :c], residual_out=bx[:, :c])
        assert torch.equal(br[:, :c], y0) and torch.equal(bx[:, :c], h0)
        wide = torch.full((9, 2 * c + 1), 7.0, device="cuda", dtype=dtype)      # two column slices that interleave
        ops.rms_norm(x, w, residual=res, out=wide[:, :c], residual_out=wide[:, c + 1:])
        assert torch.equal(wide[:, :c], y0) and torch.equal(wide[:, c + 1:], h0) and bool((wide[:, c] == 7).all())
        with pytest.raises(capi.PxeError):
            ops.rms_norm(x, w, residual=res, out=x, residual_out=x)
    img = torch.randn(2, 64, 5, 5, device="cuda").contiguous(memory_format=torch.channels_last)      # channels-last pixels are rows
    y = ops.rms_norm(img.permute(0, 2, 3, 1))[0]
    ref = img / (img.square().mean(1, keepdim=True) + 1e-6).sqrt()
    assert torch.allclose(y.permute(0, 3, 1, 2), ref, rtol=1e-5, atol=1e-6)
    for empty in (torch.empty(0, 8, device="cuda"), torch.empty(3, 0, 8, device="cuda")):
        y, h, r = ops.rms_norm(empty, residual=empty.clone())
        assert y.shape == empty.shape and r.shape == empty.shape[:-1]
        assert ops.rms_norm_e4m3(empty, group=32)[1].shape == empty.shape[:-1] + (1,)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (400, 64), (3, 1000), (333, 1023), (150, 2048), (4, 4099), (5, 8192), (2, 16384), (700, 96)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1), (2, 0)])
def test_rms_norm_backward_equals_64_bits(cuda, dtype, shape, pad, shift):
    n, c = shape
    for with_res, wtype in ((True, torch.float32), (False, dtype), (True, None)):
        h, dy = rand(13, shape, dtype, 1.0, pad, shift), rand(14, shape, dtype, 1.0, pad, shift)
        dres = rand(15, shape, dtype, 1.0, pad, shift) if with_res else None
        w = rand(16, (c,), wtype) if wtype is not None else None
        rstd = ops.rms_norm(h, w)[2]
        dx, dw = ops.rms_norm_backward(dy, h, w, rstd, dresidual=dres)
        hd, u = h.double(), dy.double() * (1.0 if w is None else w.double())
        r = rstd.double()[:, None]
        mean = (u * hd).mean(1, keepdim=True)
        dx64 = r * (u - hd * r * r * mean) + (dres.double() if with_res else 0.0)
        chain = norm_chain(c)
        spread = r * (u.abs() + hd.abs() * r * r * (u * hd).abs().mean(1, keepdim=True) * (chain + 8)) * 6 * U
        within(dx, dx64, spread + 2 * U * dx64.abs() + half_step(dtype, dx64.abs() + spread))
        if w is None:
            assert dw is None
            continue
        terms = dy.double() * hd * r
        # a column's chain: the rows of one thread, up to 8 rows of a block, the workspace's rows by 16, 16 groups
        within(dw, terms.sum(0), (n + 8 + 40 + 16 + 3) * U * terms.abs().sum(0))
        start = rand(17, (c,))
        total = start.clone()
        dx2, same = ops.rms_norm_backward(dy, h, w, rstd, dresidual=dres, dweight=total)
        assert same is total and torch.equal(dx2, dx) and torch.equal(total, start + dw)


def test_rms_norm_gradient_against_differences(cuda):
    """The sum of y * probe, differenced in 64 bits through the plain form, against dx and dweight."""
    x, res, w, probe = (rand(s, (3, 40)) for s in (18, 19, 20, 21))
    w = w[0].contiguous()
    _, h, rstd = ops.rms_norm(x, w, residual=res, eps=1e-3)
    dx, dw = ops.rms_norm_backward(probe, h, w, rstd)
    f = lambda a, b: float((norm64(a, b, None, 1e-3)[2] * probe.double()).sum())  # noqa: E731
    h64, w64, step = h.double(), w.double(), 1e-5
    for i, j in ((0, 0), (1, 17), (2, 39)):
        up, down = h64.clone(), h64.clone()
        up[i, j] += step
        down[i, j] -= step
        assert abs((f(up, w64) - f(down, w64)) / (2 * step) - float(dx[i, j])) <= 1e-5
        up, down = w64.clone(), w64.clone()
        up[j] += step
        down[j] -= step
        assert abs((f(h64, up) - f(h64, down)) / (2 * step) - float(dw[j])) <= 1e-5


def test_rms_norm_backward_in_place_and_repeatable(cuda):
    for dtype, c in ((torch.bfloat16, 768), (torch.float32, 1001), (torch.float16, 24), (torch.float32, 9001)):
        h, dy, dres, w = rand(22, (130, c), dtype), rand(23, (130, c), dtype), rand(24, (130, c), dtype), rand(25, (c,))
        rstd = ops.rms_norm(h, w)[2]
        dx, dw = ops.rms_norm_backward(dy, h, w, rstd, dresidual=dres)
        for which in range(3):
            t = [dy.clone(), h.clone(), dres.clone()]
            got, dw2 = ops.rms_norm_backward(t[0], t[1], w, rstd, dresidual=t[2], dx=t[which])
            assert got is t[which] and torch.equal(got, dx) and torch.equal(dw2, dw)
    e = torch.empty(0, 24, device="cuda")
    dx, dw = ops.rms_norm_backward(e, e.clone(), torch.ones(24, device="cuda"), torch.empty(0, device="cuda"))
    assert dx.shape == (0, 24) and bool((dw == 0).all())
    keep = torch.full((24,), 3.0, device="cuda")
    ops.rms_norm_backward(e, e.clone(), torch.ones(24, device="cuda"), torch.empty(0, device="cuda"), dweight=keep)
    assert bool((keep == 3).all())


# ------------------------------------------------------------------------------------------------ log probabilities
def probs64(x, target, temperature, top):
    """logp, entropy, top_logp, top_index of [rows, classes], from the definition in 64 bits."""
    z = x.double()
    m = z.amax(1, keepdim=True)
    d = (z - torch.where(m == -INF, torch.zeros_like(m), m)) / temperature
    e = d.exp()
    total = e.sum(1)
    lp = torch.where((total == 0)[:, None], torch.full_like(d, -INF), d - total.log()[:, None])
    h = total.log() - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1) / total
    h = torch.where(total == 0, torch.zeros_like(h), h)
    out = [None, h, None, None]
    if target is not None:
        out[0] = lp.gather(1, target.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0]
        out[0] = torch.where(target >= x.shape[1], torch.full_like(h, NAN), out[0])
    if top:
        order = torch.where(z.isnan(), torch.full_like(z, INF), z)             # a NaN above every number
        first = z.isnan().double()
        index = torch.argsort(-order, dim=1, stable=True)
        index = index.gather(1, torch.argsort(-first.gather(1, index), dim=1, stable=True))[:, :top]
        out[2], out[3] = lp.gather(1, index), index.int()
    if target is not None:
        gone = target < 0
        out[0] = out[0].masked_fill(gone, 0)
        out[1] = out[1].masked_fill(gone, 0)
        if top:
            out[2], out[3] = out[2].masked_fill(gone[:, None], 0), out[3].masked_fill(gone[:, None], -1)
    return out, lp


def probs_tol(v, h, logp):
    """Sums of up to v / 512 + 40 additions, terms of eight roundings and an exponential (2 units of 2^-23) at up to 40
    from the maximum; what a logarithm and a difference of this size round to."""
    return U * ((v / 512 + 40) + 150) * (1 + math.log(v + 1) + h.abs()) + 6 * U * logp.abs()


def check_probs(x, target, temperature=1.0, top=0):
    r = ops.log_probs(x, target, top=top, temperature=temperature)
    x2 = x.reshape(-1, x.shape[-1])
    t2 = None if target is None else target.reshape(-1)
    (logp, h, top_logp, top_index), lp = probs64(x2, t2, temperature, top)
    tol_h = torch.nan_to_num(h)
    v = x2.shape[1]
    within(r.entropy.reshape(-1), h, probs_tol(v, tol_h, tol_h))
    if target is not None:
        fine = torch.nan_to_num(logp, nan=0.0, neginf=0.0)
        within(r.logp.reshape(-1), logp, probs_tol(v, tol_h, fine))
    else:
        assert r.logp is None
    if top:
        assert torch.equal(r.top_index.reshape(-1, top), top_index)
        fine = torch.nan_to_num(top_logp, nan=0.0, neginf=0.0)
        within(r.top_logp.reshape(-1, top), top_logp, probs_tol(v, tol_h[:, None], fine))
    else:
        assert r.top_logp is None and r.top_index is None
    return r, lp


PROB_SHAPES = [(1, 1), (3, 2), (5, 31), (64, 80), (2, 1000), (3, 1023), (200, 33), (1, 4096), (2, 8193), (5, 32000), (2, 50003), (1, 131072), (1, 262147)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", PROB_SHAPES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1), (8, 0)])
def test_log_probs_equal_64_bits(cuda, dtype, shape, pad, shift):
    n, v = shape
    x = rand(30, shape, dtype, 3.0, pad, shift)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen(31))
    check_probs(x, target)
    check_probs(x, target.int(), temperature=0.6, top=min(20, v))
    check_probs(x, None, temperature=2.5, top=min(1, v))
    if n > 2:
        target[1] = -100
        check_probs(x, target, top=min(32, v))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [5, 40, 1500, 9001, 70000])
def test_log_probs_masked_and_extreme_rows(cuda, dtype, v):
    info = torch.finfo(dtype)
    x = rand(32, (12, v), dtype, 2.0)
    x[0] = -INF                                           # nothing left
    x[1] = -INF
    x[1, v - 1] = 0.5                                     # one left
    x[2] = info.min                                       # lowest throughout: uniform
    x[3] = info.min
    x[3, 2] = 1.0                                         # masked with the lowest value
    x[4, 0] = -INF
    x[5, v // 2] = NAN
    x[6, 1] = INF
    x[7] = info.max
    x[8] = 0.0                                            # all equal: ties to the lower class
    x[8, 1] = -0.0
    x[9, 1:] = -INF
    x[9, 0] = info.min
    x[10] = torch.arange(v, device="cuda").to(dtype) % 7
    x[11] = torch.linspace(-300, 300, v, device="cuda").to(dtype)
    target = torch.tensor([0, v - 1, 1, 2, 0, 1, 0, 3, 1, 0, 4, v - 1], device="cuda")
    finite = [0, 1, 2, 3, 4, 7, 8, 9, 10, 11]
    for temperature in (1.0, 0.5):
        r, _ = check_probs(x[finite], target[finite], temperature, top=min(5, v))
    assert float(r.logp[0]) == -INF and float(r.entropy[0]) == 0 and r.top_index[0].tolist() == list(range(5))
    assert float(r.logp[1]) == 0 and float(r.entropy[1]) == 0
    r = ops.log_probs(x[5:7], target[5:7], top=2)
    assert bool(r.logp.isnan().all()) and bool(r.entropy.isnan().all()) and bool(r.top_logp.isnan().all())
    assert r.top_index[:, 0].tolist() == [v // 2, 1]
    # the gradient of the same rows: finite where the row is, zero where nothing is left
    full = ops.log_probs(x, target)
    ones = torch.ones(12, device="cuda")
    dx = ops.log_probs_backward(x, target, full.stats, ones, dentropy=ones)
    assert bool((dx[0] == 0).all()) and bool((dx[1] == 0).all())
    broken = (x.isnan() | (x == INF)).any(1)              # row 10 too where its type ends before 70000
    assert bool(dx[~broken].isfinite().all()) and bool(dx[broken].isnan().any(1).all()) and bool(broken[5] & broken[6])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [7, 3000, 80001])
@pytest.mark.parametrize("temperature", [1e-8, 0.01, 50.0, 100.0, 1e6])
def test_log_probs_at_extreme_temperatures(cuda, dtype, v, temperature):
    """-inf stays without weight and the type's lowest value keeps the one it has, whatever the temperature; values of the
    order of the temperature, so that something is left to compare."""
    info = torch.finfo(dtype)
    x = rand(45, (6, v), dtype, min(2.0 * temperature, 1e4))
    x[1, 1::2] = -INF
    x[2] = info.min
    x[2, ::3] = -INF
    x[3] = -INF
    x[3, v - 1] = info.min
    x[4, 2:] = info.min
    x[5, 1:] = -INF
    target = torch.tensor([1, 0, 1, v - 1, 0, 0], device="cuda")
    check_probs(x, target, temperature, top=min(9, v))


def test_log_probs_many_large_values_with_one_thread(cuda):
    """Ascending, descending and strided rows, where the largest values lie close together or all belong to elements that
    one thread takes (every 4096th vector and the like): the list of candidates runs over."""
    for dtype in TYPES:
        v = 1 << 18
        x = torch.full((4, v), -1.0, device="cuda", dtype=dtype)
        x[0] = torch.arange(v, device="cuda").to(dtype) * 2 ** -10
        x[1] = -torch.arange(v, device="cuda").to(dtype) * 2 ** -10
        per = 16 // x.element_size()
        for step in (512 * per, 256 * per, 1024 * per):
            x[2] = -1.0
            for k in range(32):                           # 32 threads that hold nothing but large values
                for j in range(per):
                    at = torch.arange(k * per + j, v, step, device="cuda")
                    x[2, at] = (1.0 + torch.arange(len(at), device="cuda") % 50 / 64).to(dtype)
            x[3] = x[2].flip(0)
            check_probs(x, None, top=32)
            check_probs(x, None, top=7)


def test_log_probs_slices_and_padding(cuda):
    x = rand(33, (3, 9, 101), torch.bfloat16, 2.0)
    target = torch.randint(0, 101, (3, 9), device="cuda", generator=gen(34))
    target[1, 4:] = -1                                    # a padded sequence
    whole = ops.log_probs(x[:, :-1].contiguous(), target[:, 1:].contiguous(), top=3)
    part = ops.log_probs(x[:, :-1], target[:, 1:].contiguous(), top=3)
    assert torch.equal(whole.top_index, part.top_index)
    for a, b in zip(whole, part):                         # a row's place decides which thread sums what: each is within the tolerance
        if a.dtype == torch.float32:
            within(a, b, 2 * probs_tol(101, torch.full_like(b.double(), math.log(101)), b.double()))
    d = rand(35, (3, 8))
    keep = x.clone()
    dx = ops.log_probs_backward(x[:, :-1], target[:, 1:].contiguous(), part.stats, d)
    want = ops.log_probs_backward(x[:, :-1].contiguous(), target[:, 1:].contiguous(), part.stats, d)
    assert torch.equal(dx, want)
    ops.log_probs_backward(x[:, :-1], target[:, 1:].contiguous(), part.stats, d, dx=x[:, :-1])      # in place on a slice
    assert torch.equal(x[:, :-1], want) and torch.equal(x[:, -1], keep[:, -1])
    buf = torch.full((3, 8, 107), 7.0, device="cuda", dtype=torch.bfloat16)                        # another distance from a boundary
    ops.log_probs_backward(keep[:, :-1], target[:, 1:].contiguous(), part.stats, d, dx=buf[..., 3:104])
    assert torch.equal(buf[..., 3:104], want) and bool((buf[..., :3] == 7).all()) and bool((buf[..., 104:] == 7).all())
    both = torch.full((3, 9, 202), 7.0, device="cuda", dtype=torch.bfloat16)                       # columns of one buffer, and rows of one
    both[..., :101] = keep
    ops.log_probs_backward(both[:, :-1, :101], target[:, 1:].contiguous(), part.stats, d, dx=both[:, :-1, 101:])
    assert torch.equal(both[:, :-1, 101:], want) and torch.equal(both[..., :101], keep) and bool((both[:, -1, 101:] == 7).all())
    long = torch.zeros((3, 16, 101), device="cuda", dtype=torch.bfloat16)
    long[:, :8] = keep[:, :-1]
    ops.log_probs_backward(long[:, :8], target[:, 1:].contiguous(), part.stats, d, dx=long[:, 8:])
    assert torch.equal(long[:, 8:], want)
    e = ops.log_probs(torch.empty(0, 7, device="cuda"), torch.empty(0, device="cuda", dtype=torch.int64), top=2)
    assert e.logp.shape == (0,) and e.top_index.shape == (0, 2)
    r = ops.log_probs(rand(36, (3, 50)), torch.tensor([1, 50, 1 << 40], device="cuda"))             # classes that are not there
    assert r.logp.isnan().tolist() == [False, True, True] and bool(r.entropy.isfinite().all())
    assert float(ops.log_probs(rand(37, (9,)), torch.tensor(3, device="cuda")).logp) < 0            # a single row


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (4, 3), (300, 80), (5, 1000), (3, 4097), (2, 50003), (33, 8192)])
@pytest.mark.parametrize("pad", [0, 1])
def test_log_probs_backward_equals_64_bits(cuda, dtype, shape, pad):
    n, v = shape
    x = rand(38, shape, dtype, 2.0, pad)
    if v > 10:
        x[:, 3:6] = -INF
    target = torch.randint(0, v, (n,), device="cuda", generator=gen(39))
    target = torch.where((target >= 3) & (target < 6) & (v > 10), torch.zeros_like(target), target)
    if n > 2:
        target[2] = -1
    dlogp, dh = rand(40, (n,)), rand(41, (n,))
    for temperature in (1.0, 0.7):
        r = ops.log_probs(x, target, temperature=temperature)
        (_, h, _, _), lp = probs64(x, target, temperature, 0)
        p = lp.exp()
        lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
        used = (target >= 0).double()[:, None]
        hot = torch.zeros_like(p).scatter_(1, target.clamp(min=0)[:, None], 1.0)
        for g, gh in ((dlogp, None), (None, dh), (dlogp, dh)):
            dx = ops.log_probs_backward(x, target, r.stats, g, dentropy=gh, temperature=temperature)
            assert dx.stride() == x.stride()
            gd = torch.zeros(n, 1, dtype=torch.float64, device="cuda") if g is None else g.double()[:, None]
            hd = torch.zeros(n, 1, dtype=torch.float64, device="cuda") if gh is None else gh.double()[:, None]
            want = used * (gd * (hot - p) - hd * p * (lp0 + h[:, None])) / temperature
            size = (gd.abs() * (hot + p) + hd.abs() * p * (lp0.abs() + h[:, None].abs() + math.log(v + 1) + 1)) / temperature
            tol = size * U * ((v / 512 + 40) + 200)
            within(dx, want, tol + half_step(dtype, want.abs() + tol) + 1e-37)
            again = x.clone(memory_format=torch.preserve_format)
            assert torch.equal(ops.log_probs_backward(again, target, r.stats, g, dentropy=gh, temperature=temperature, dx=again), dx)


def test_log_probs_gradient_against_differences(cuda):
    x, dlogp, dh = rand(42, (3, 30), torch.float32, 2.0), rand(43, (3,)), rand(44, (3,))
    target = torch.tensor([4, 0, 29], device="cuda")
    r = ops.log_probs(x, target, temperature=1.3)
    dx = ops.log_probs_backward(x, target, r.stats, dlogp, dentropy=dh, temperature=1.3)

    def f(a):
        (logp, h, _, _), _ = probs64(a, target, 1.3, 0)
        return float((logp * dlogp.double() + h * dh.double()).sum())
    step = 1e-5
    for i, j in ((0, 4), (0, 5), (1, 0), (2, 11)):
        up, down = x.double(), x.double()
        up[i, j] += step
        down[i, j] -= step
        assert abs((f(up) - f(down)) / (2 * step) - float(dx[i, j])) <= 1e-5


# ------------------------------------------------------------------------------------------------ AdamW
def make_params(seed, sizes, dtype, shift=0):
    """Tensors in one buffer, `shift` elements off a 256-byte boundary each."""
    return [rand(seed + k, (n + shift,), dtype, 0.05)[shift:] for k, n in enumerate(sizes)]


def adamw64(p, g, m, v, t, rate, b1, b2, eps, wd, gs):
    g = g.double() * gs
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = (v1 / (1 - b2 ** t)).sqrt() + eps
    p1 = p - rate * ((m1 / (1 - b1 ** t)) / den + wd * p)
    m_tol = 4 * U * (b1 * m.abs() + (1 - b1) * g.abs())
    p_tol = rate * (m_tol / (1 - b1 ** t) / den + 16 * U * (m1 / (1 - b1 ** t) / den).abs() + 4 * U * (wd * p).abs()) + 2 * U * p1.abs()
    return p1, m1, v1, p_tol, m_tol


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


SIZES = [1, 255, 256, 257, 3, 4096, 10007, 8192 + 256, 0, 100000]


@pytest.mark.parametrize("dtype,gtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
                                         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                         (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_steps_equal_64_bits(cuda, dtype, gtype, bits, master, shift):
    if master and dtype == torch.float32:
        with pytest.raises(ValueError):
            ops.AdamW([torch.zeros(4, device="cuda")], master=True)
        return
    params = make_params(100, SIZES, dtype, shift)
    plan = ops.AdamW(params, state_bits=bits, master=master)
    hyper = dict(rate=1e-2, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1, grad_scale=0.5)
    rate, b1, b2, eps, wd, gs = (f32(v) for v in hyper.values())
    blocks = [-(-n // 256) for n in SIZES]

    def state():
        if bits == 32:
            return [m.double() for m in plan.m], [v.double() for v in plan.v]
        wide = lambda q, s: q.double() * s.double().repeat_interleave(256)[:q.numel()]  # noqa: E731
        return [wide(q, s) for q, s in zip(plan.m, plan.m_scale)], [wide(q, s).square() for q, s in zip(plan.v, plan.v_scale)]

    for t in (1, 2, 3):
        m0, v0 = state()
        p0 = [(plan.master[k] if master else p).double().clone() for k, p in enumerate(params)]
        grads = make_params(200 + 20 * t, SIZES, gtype, shift)
        if t == 2:
            for g in grads:
                g.zero_()
        plan.step(grads, t=t, **hyper)
        for k in range(len(SIZES)):
            if SIZES[k] == 0:
                continue
            p1, m1, v1, p_tol, m_tol = adamw64(p0[k], grads[k], m0[k], v0[k], t, rate, b1, b2, eps, wd, gs)
            if master:
                within(plan.master[k], p1, p_tol)
                assert torch.equal(params[k], plan.master[k].to(dtype))
            else:
                within(params[k], p1, p_tol + half_step(dtype, p1.abs() + p_tol))
            if bits == 32:
                within(plan.m[k], m1, m_tol)
                within(plan.v[k], v1, 6 * U * v1)
                continue
            for q, s, want, off in ((plan.m[k], plan.m_scale[k], m1, m_tol), (plan.v[k], plan.v_scale[k], v1.sqrt(), 6 * U * v1.sqrt())):
                wide = torch.zeros(blocks[k] * 256, dtype=torch.float64, device="cuda")
                wide[:SIZES[k]] = want
                big = wide.view(-1, 256).abs().amax(1)
                within(s, (big / 448).clamp(min=2.0 ** -126), big / 448 * 16 * U + 1e-45)
                each = s.double().repeat_interleave(256)[:SIZES[k]]
                # half a step of a code: 2^-4 of the value, 2^-10 of the scale among the smallest
                tol = want.abs() * (2.0 ** -4 * 1.001) + each * 2.0 ** -10 * 1.001 + 2 * off
                if q is plan.v[k]:
                    tol = tol + torch.where(want > 0, each * 2.0 ** -10 * 1.001, torch.zeros_like(each))   # never below the smallest code
                    assert bool(((q.float() > 0) == (want > 0)).all())
                within(q.double() * each, want, tol)


def test_adamw_many_tensors_and_repeatable(cuda):
    """More tensors than one launch takes; each gets what it gets alone; twice the same bits."""
    sizes = [(37 * k) % 700 + 1 for k in range(900)]
    params, grads = make_params(1000, sizes, torch.float32), make_params(3000, sizes, torch.float32)
    runs = []
    for _ in range(2):
        mine = [p.clone() for p in params]
        plan = ops.AdamW(mine)
        for t in (1, 2):
            plan.step(grads, rate=1e-3, t=t, weight_decay=0.01)
        runs.append((mine, plan))
    for k in range(900):
        assert torch.equal(runs[0][0][k], runs[1][0][k]) and torch.equal(runs[0][1].v[k], runs[1][1].v[k])
    for k in (0, 399, 400, 401, 799, 800, 899):
        alone = [params[k].clone()]
        plan = ops.AdamW(alone)
        for t in (1, 2):
            plan.step([grads[k]], rate=1e-3, t=t, weight_decay=0.01)
        assert torch.equal(alone[0], runs[0][0][k])


def test_adamw_device_scalars_skip_and_graph(cuda):
    """rate, t and grad_scale from device memory give what the numbers give (to the rounding of 1 - beta^t); a captured
    step reads the current ones; a skip flag leaves every bit."""
    sizes = [1000, 77, 4096]
    for bits in (32, 8):
        grads = make_params(50, sizes, torch.float32)
        a, b = make_params(60, sizes, torch.float32), make_params(60, sizes, torch.float32)
        pa, pb = ops.AdamW(a, state_bits=bits), ops.AdamW(b, state_bits=bits)
        rate, t, gs = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int64), torch.ones(1, device="cuda")
        skip = torch.zeros(1, device="cuda")
        skip.fill_(1.0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            pb.step(grads, rate=rate, t=t, grad_scale=gs, skip=skip)
            with torch.cuda.graph(graph, stream=side):
                pb.step(grads, rate=rate, t=t, grad_scale=gs, skip=skip)
        torch.cuda.current_stream().wait_stream(side)
        before = [x.clone() for x in b + pb.m + pb.v]
        graph.replay()
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(b + pb.m + pb.v, before))
        skip.zero_()
        for step, (r, s) in enumerate(((1e-3, 1.0), (2e-3, -0.5), (1e-4, 3.0)), start=1):
            rate.fill_(r)
            t.fill_(step)
            gs.fill_(s)
            graph.replay()
            pa.step(grads, rate=r, t=step, grad_scale=s)
            for x, y in zip(a, b):
                # an update of at most rate * 10 here; 1 - beta^t of both kinds agree to 8 units
                assert float((x - y).abs().max()) <= 10 * r * 16 * U + 2 * U * float(x.abs().max())
            if bits == 32:
                assert all(torch.equal(x, y) for x, y in zip(pa.m + pa.v, pb.m + pb.v))


def test_adamw_non_finite_gradients_stay_where_they_are(cuda):
    n = 3000
    for bits in (32, 8):
        p = make_params(70, [n], torch.float32)
        clean = [p[0].clone()]
        g = make_params(71, [n], torch.float32)
        plan, ref = ops.AdamW(p, state_bits=bits), ops.AdamW(clean, state_bits=bits)
        ref.step(g, rate=1e-3, t=1)
        bad = g[0].clone()
        bad[700] = NAN
        bad[2999] = INF
        plan.step([bad], rate=1e-3, t=1)
        ok = torch.ones(n, dtype=torch.bool, device="cuda")
        ok[700] = ok[2999] = False
        assert torch.equal(p[0][ok], clean[0][ok]) and bool(p[0][~ok].isnan().all())
        lost = ~ok if bits == 32 else torch.zeros(n, dtype=torch.bool, device="cuda")
        if bits == 8:
            lost[512:768] = lost[2816:] = True
        assert torch.equal(plan.m[0].float()[~lost], ref.m[0].float()[~lost])


def test_adamw_state_is_adopted_and_moved_parameters_refused(cuda):
    sizes = [300, 50]
    for bits in (32, 8):
        a, grads = make_params(80, sizes, torch.bfloat16), make_params(90, sizes, torch.bfloat16)
        b = [p.clone() for p in a]
        one = ops.AdamW(a, state_bits=bits, master=True)
        one.step(grads, rate=1e-2, t=1)
        copy = lambda ts: None if ts is None else [t.clone() for t in ts]  # noqa: E731
        for x, y in zip(b, a):
            x.copy_(y)
        two = ops.AdamW(b, state_bits=bits, m=copy(one.m), v=copy(one.v), m_scale=copy(one.m_scale), v_scale=copy(one.v_scale), master=copy(one.master))
        one.step(grads, rate=1e-2, t=2)
        two.step(grads, rate=1e-2, t=2)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        with pytest.raises(ValueError):
            two.step(grads[:1], rate=1e-2, t=3)
        with pytest.raises(ValueError):
            two.step([grads[0], grads[1][:49]], rate=1e-2, t=3)
        with pytest.raises(ValueError):
            two.step([grads[0], grads[1].float()], rate=1e-2, t=3)
        with pytest.raises(TypeError):
            two.step([grads[0], None], rate=1e-2, t=3)
        with pytest.raises(capi.PxeError):
            two.step([g.half() for g in grads], rate=1e-2, t=3)
        with pytest.raises(capi.PxeError):
            two.step(grads, rate=1e-2, t=0)
        b[0].data = b[0].data.clone()
        with pytest.raises(RuntimeError):
            two.step(grads, rate=1e-2, t=3)
    p = torch.zeros(8, device="cuda")
    with pytest.raises(capi.PxeError):
        ops.AdamW([p, p]).step([p.clone(), p.clone()], rate=1e-3, t=1)
    with pytest.raises(TypeError):
        ops.AdamW([p, p.half()])
    with pytest.raises(ValueError):
        ops.AdamW([torch.zeros(4, 4, device="cuda").t()])
    with pytest.raises(ValueError):
        ops.AdamW([p], m=[p.clone()])
    with pytest.raises(ValueError):
        ops.AdamW([p], state_bits=8, m=[p.clone()], v=[p.clone()])


# ------------------------------------------------------------------------------------------------ together
def test_a_training_step_of_the_three_together(cuda):
    """Residual, norm, classifier, log probabilities with an entropy term, all gradients and an AdamW step, twice, against
    the same in 64 bits through autograd."""
    n, c, v = 96, 200, 130
    x, res = rand(400, (n, c)), rand(401, (n, c))
    weight, head = 1 + 0.1 * rand(402, (c,)), rand(403, (v, c), scale=0.1)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen(404))
    target[5] = -1
    params = [weight.clone(), head.clone(), x.clone()]
    plan = ops.AdamW(params)
    ref = [p.double().requires_grad_(True) for p in params]
    opt = torch.optim.AdamW(ref, lr=f32(1e-2), betas=(f32(0.9), f32(0.999)), eps=f32(1e-8), weight_decay=f32(0.1))
    dlogp = torch.where(target >= 0, -1.0 / 95, 0.0).float()
    dentropy = torch.where(target >= 0, -0.05 / 95, 0.0).float()
    for t in (1, 2):
        y, h, rstd = ops.rms_norm(params[2], params[0], residual=res)
        logits = y @ params[1].t()
        r = ops.log_probs(logits, target)
        dlogits = ops.log_probs_backward(logits, target, r.stats, dlogp, dentropy=dentropy)
        dx, dweight = ops.rms_norm_backward(dlogits @ params[1], h, params[0], rstd)
        dhead = dlogits.t() @ y
        opt.zero_grad()
        hd = ref[2] + res.double()
        yd = hd * torch.rsqrt(hd.square().mean(1, keepdim=True) + 1e-6) * ref[0]
        lp = torch.log_softmax(yd @ ref[1].t(), 1)
        logp = lp.gather(1, target.clamp(min=0)[:, None])[:, 0]
        loss = (logp * dlogp.double() - (lp.exp() * lp).sum(1) * dentropy.double()).sum()
        loss.backward()
        for got, want in ((dweight, ref[0].grad), (dhead, ref[1].grad), (dx, ref[2].grad)):
            # products of 130 to 200 terms in 32 bits (no reduced-precision products) after a dozen roundings
            assert float((got.double() - want).abs().max()) <= 300 * U * float(want.abs().max()) + 1e-9
        # the first steps divide m by |m|: the parameters take the exact gradients, so that both sides step alike
        plan.step([ref[0].grad.float(), ref[1].grad.float(), ref[2].grad.float()], rate=1e-2, t=t, weight_decay=0.1)
        opt.step()
        for got, want in zip(params, ref):
            assert float((got.double() - want.detach()).abs().max()) <= 1e-2 * 200 * U + 4 * U * float(want.detach().abs().max())
            with torch.no_grad():
                want.copy_(got.double())


def test_served_answer_of_the_two_together(cuda):
    """Norm with 8-bit output, the product of what the codes stand for, and the alternatives; captured once and replayed on
    new inputs, with the bits of the eager calls."""
    n, c, v = 3, 512, 4001
    x, res, w, head = rand(410, (n, c), torch.bfloat16), rand(411, (n, c), torch.bfloat16), rand(412, (c,)), rand(413, (v, c), torch.bfloat16, 0.1)

    def answer():
        q, scale, h, rstd = ops.rms_norm_e4m3(x, w, residual=res, group=128)
        y = (q.float() * scale.repeat_interleave(128, 1)).bfloat16()
        return (q.view(torch.uint8), scale, h, rstd) + tuple(t for t in ops.log_probs(y @ head.t(), top=5, temperature=0.8) if t is not None)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        answer()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = answer()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (420, 421):
        x.copy_(rand(seed, (n, c), torch.bfloat16))
        graph.replay()
        for a, b in zip(held, answer()):
            assert torch.equal(a, b)


def test_two_streams_at_once(cuda):
    """The backward pass of two threads' worth of streams, each with its own workspace: the bits of one after the other."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    data = [(rand(430 + k, (500, 1536), torch.bfloat16), rand(440 + k, (500, 1536), torch.bfloat16)) for k in range(2)]
    w = rand(450, (1536,))
    want = []
    for h, dy in data:
        rstd = ops.rms_norm(h, w)[2]
        want.append((rstd,) + ops.rms_norm_backward(dy, h, w, rstd))
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, (h, dy), (rstd, _, _) in zip((a, b), data, want):
            with torch.cuda.stream(s):
                got.append(ops.rms_norm_backward(dy, h, w, rstd))
        torch.cuda.synchronize()
        for (dx, dw), (_, dx0, dw0) in zip(got, want):
            assert torch.equal(dx, dx0) and torch.equal(dw, dw0)


def test_rows_beyond_32_bits(cuda):
    """Rows more than 2^30 elements apart (offsets past 2^31), and a parameter of more than 2^31 elements: what lies there is
    what the same rows and blocks give on their own."""
    big = torch.zeros((1 << 31) + 8192, device="cuda", dtype=torch.bfloat16)
    stride = (1 << 30) + 8
    x, y = big.as_strided((3, 1000), (stride, 1)), big.as_strided((3, 1000), (stride, 1), 2048)
    x.copy_(rand(500, (3, 1000), torch.bfloat16))
    dense = x.contiguous()
    w, target = rand(501, (1000,)), torch.tensor([5, 999, 0], device="cuda")
    want, _, rstd = ops.rms_norm(dense, w)
    ops.rms_norm(x, w, out=y)
    assert torch.equal(y, want)
    ops.rms_norm_backward(x, x, w, rstd, dx=y)
    assert torch.equal(y, ops.rms_norm_backward(dense, dense, w, rstd)[0])
    far, near = ops.log_probs(x, target, top=3), ops.log_probs(dense, target, top=3)
    assert all(torch.equal(a, b) for a, b in zip(far, near))
    d = rand(502, (3,))
    ops.log_probs_backward(x, target, far.stats, d, dx=y)
    assert torch.equal(y, ops.log_probs_backward(dense, target, near.stats, d))
    del x, y
    n = big.numel() - 5                                   # the last block is short
    param, grad = big[:n], torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16)
    tail = slice(n // 256 * 256 - 1024, n)
    param[tail] = rand(503, (n - tail.start,), torch.bfloat16)
    grad[tail] = rand(504, (n - tail.start,), torch.bfloat16)
    small = [param[tail].clone()]
    plan, alone = ops.AdamW([param], state_bits=8), ops.AdamW(small, state_bits=8)
    plan.step([grad], rate=1e-2, t=1)
    alone.step([grad[tail].clone()], rate=1e-2, t=1)
    assert torch.equal(param[tail], small[0]) and torch.equal(plan.m[0][tail].view(torch.uint8), alone.m[0].view(torch.uint8))
    assert torch.equal(plan.v_scale[0][-5:], alone.v_scale[0]) and bool((big[n:] == 0).all())
    assert bool((param[4000:9000] == param[4000]).all()) and float(param[4000]) != 0            # (zeros before the step)


def test_many_rows_of_few_classes(cuda):
    x = rand(510, (70001, 3), torch.float16)
    target = torch.randint(-1, 3, (70001,), device="cuda", generator=gen(511))
    r, _ = check_probs(x, target, top=2)
    d = rand(512, (70001,))
    dx = ops.log_probs_backward(x, target, r.stats, d)
    p = torch.softmax(x.double(), 1)
    hot = torch.nn.functional.one_hot(target.clamp(min=0), 3).double()
    want = (target >= 0).double()[:, None] * d.double()[:, None] * (hot - p)
    within(dx, want, 64 * U * d.abs().double()[:, None] + half_step(torch.float16, want))
    y, _, rstd = ops.rms_norm(x)
    f = x.double()
    r64 = 1 / (f.square().mean(1) + 1e-6).sqrt()
    within(rstd, r64, r64 * 8 * U)
    within(y, f * r64[:, None], (f * r64[:, None]).abs() * 10 * U + half_step(torch.float16, f * r64[:, None]))


def test_a_captured_training_step_equals_the_eager_one(cuda):
    """Norm, log probabilities, both gradients and the step captured in one graph, with t on the device, replayed on new
    inputs: the bits of the eager calls (the weight gradient's second launch included)."""
    n, c, v = 700, 1024, 511
    x, res, head = rand(520, (n, c), torch.bfloat16), rand(521, (n, c), torch.bfloat16), rand(522, (v, c), torch.bfloat16, 0.1)
    target, dlogp = torch.randint(0, v, (n,), device="cuda", generator=gen(523)), rand(524, (n,))
    t = torch.zeros(1, device="cuda", dtype=torch.int64)

    def step(weight, plan):
        y, h, rstd = ops.rms_norm(x, weight, residual=res)
        logits = y @ head.t()
        r = ops.log_probs(logits, target)
        dlogits = ops.log_probs_backward(logits, target, r.stats, dlogp, dx=logits)
        dx, dweight = ops.rms_norm_backward(dlogits @ head, h, weight, rstd, dresidual=h)
        plan.step([dweight], rate=1e-3, t=t, weight_decay=0.01)
        return r.logp, dx, dweight

    a, b = rand(525, (c,)), rand(525, (c,))
    pa, pb = ops.AdamW([a]), ops.AdamW([b])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = rand(526, (c,))
        step(warm, ops.AdamW([warm]))                     # (t is 0 here and its result is not looked at)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step(b, pb)
    torch.cuda.current_stream().wait_stream(side)
    for k in (1, 2, 3):
        x.copy_(rand(530 + k, (n, c), torch.bfloat16))
        t.fill_(k)
        graph.replay()
        for got, want in zip(held, step(a, pa)):
            assert torch.equal(got, want)
        assert torch.equal(a, b) and torch.equal(pa.m[0], pb.m[0]) and torch.equal(pa.v[0], pb.v[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1030, 2000, 2051, 4100, 8190, 16383])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1)])
def test_log_probs_of_many_rows_of_middling_length(cuda, dtype, v, pad, shift):
    """Rows enough to fill the card, which are read by fewer threads each: a thread of the fewest adds v / 128 terms (to each
    of two halves), a lane of a warp up to 64; both are under the v / 64 + 40 of a row eight times as long."""
    n, info = 1300, torch.finfo(dtype)
    x = rand(52, (n, v), dtype, 2.0, pad, shift)
    x[0] = -INF                                           # nothing left
    x[1] = -INF
    x[1, v - 1] = 0.5                                     # one left
    x[2] = info.min
    x[3, 5:] = info.min
    x[4] = info.max
    x[5] = 0.0                                            # ties throughout
    x[6] = torch.arange(v, device="cuda").to(dtype) % 7
    x[7, 100:] = -INF
    x[8, : v // 2] = 6.0                                  # more ties than any list holds
    x[n - 1] = torch.linspace(-300, 300, v, device="cuda").to(dtype)
    x[20:40, ::2] = -INF
    target = torch.randint(0, v, (n,), device="cuda", generator=gen(53))
    target[0], target[1] = 0, v - 1
    target[50:90] = -1
    target[n - 2] = -100
    target[91] = v
    for top, temperature in ((0, 1.0), (1, 0.7), (32, 1.0)):
        r = ops.log_probs(x, target, top=top, temperature=temperature)
        (logp, h, top_logp, top_index), _ = probs64(x, target, temperature, top)
        tol = lambda want: probs_tol(8 * v, h if want.dim() == 1 else h[:, None], torch.nan_to_num(want, nan=0.0, neginf=0.0))  # noqa: E731
        within(r.entropy, h, tol(h))
        within(r.logp, logp, tol(logp))
        if top:
            assert torch.equal(r.top_index, top_index)
            within(r.top_logp, top_logp, tol(top_logp))
    x[9, v // 2], x[10, 1] = NAN, INF
    r = ops.log_probs(x[9:11], top=2)
    many = ops.log_probs(x, target.clamp(0, v - 1), top=2)
    for got in (r, many._replace(logp=None, entropy=many.entropy[9:11], top_logp=many.top_logp[9:11], top_index=many.top_index[9:11])):
        assert bool(got.entropy.isnan().all()) and bool(got.top_logp.isnan().all()) and got.top_index[:, 0].tolist() == [v // 2, 1]
    assert bool(many.logp[9:11].isnan().all()) and bool(many.entropy[11:].isfinite().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [130, 1025, 2047, 4096, 4111, 9000])
def test_log_probs_gradient_of_rows_in_parts(cuda, dtype, v):
    """Rows of one part and of several, whole vectors and single elements (where dx lies otherwise than x)."""
    n = 37
    x = rand(54, (n, v), dtype, 2.0, 3, 1)
    target = torch.randint(-1, v, (n,), device="cuda", generator=gen(55))
    d = rand(56, (n,))
    r = ops.log_probs(x, target)
    (_, h, _, _), lp = probs64(x, target, 1.0, 0)
    hot = torch.zeros_like(lp).scatter_(1, target.clamp(min=0)[:, None], 1.0)
    g = d.double()[:, None] * (target >= 0).double()[:, None]
    want, size = g * (hot - lp.exp()), g.abs() * (hot + lp.exp())
    tol = size * U * ((v / 64 + 40) + 200)
    for dx in (None, torch.empty(n, v, device="cuda", dtype=dtype), torch.empty(n, v + 5, device="cuda", dtype=dtype)[:, 2:v + 2]):
        got = ops.log_probs_backward(x, target, r.stats, d, dx=dx)
        within(got, want, tol + half_step(dtype, want.abs() + tol) + 1e-37)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(1, 1), (15, 3), (16, 7), (17, 31), (1000, 32), (33, 40), (1001, 80), (50, 127), (19, 128), (65, 200), (31, 257), (15, 263)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1), (5, 3)])
def test_log_probs_of_short_rows(cuda, dtype, n, v, pad, shift):
    """Rows that share a warp, with their gradient: masked ones, unused ones and a last warp that is not full."""
    x = rand(57, (n, v), dtype, 2.0, pad, shift)
    x[n // 2] = -INF
    x[n // 3, 1:] = -INF
    if n > 8:
        x[2] = torch.finfo(dtype).min
        x[3] = 0.0
        x[7, v - 1] = -INF
    target = torch.randint(0, v, (n,), device="cuda", generator=gen(58))
    target[n // 2] = 0
    check_probs(x, None, temperature=0.5)
    check_probs(x, target.int())
    target[n // 4::5] = -1
    if n > 8:
        target[6] = v
    r, lp = check_probs(x, target, temperature=1.5)
    assert torch.equal(r.stats[target < 0], torch.zeros_like(r.stats[target < 0]))
    target = target.clamp(max=v - 1)
    d = rand(59, (n,))
    used = ((target >= 0) & (x != -INF).any(1)).double()[:, None]
    p = torch.nan_to_num(lp, neginf=-1e9).exp()
    hot = torch.zeros_like(p).scatter_(1, target.clamp(min=0)[:, None], 1.0)
    size = used * d.double()[:, None].abs() * (hot + p) / 1.5
    want = used * d.double()[:, None] * (hot - p) / 1.5
    tol = size * U * ((v / 512 + 40) + 200)
    within(ops.log_probs_backward(x, target, r.stats, d, temperature=1.5), want, tol + half_step(dtype, want.abs() + tol) + 1e-37)
    if n > 8:
        wide = x[6:n - n % 2].reshape(2, -1, v)[:, 1:]     # groups of rows, where they lie
        a, b = ops.log_probs(wide), ops.log_probs(wide.contiguous())
        within(a.entropy, b.entropy, 2 * probs_tol(v, torch.nan_to_num(b.entropy), torch.nan_to_num(b.entropy)))
    if n > 20:
        x[11, v // 2], x[12, 0] = NAN, INF
        r = ops.log_probs(x, target.clamp(min=0))
        assert bool(r.logp[11:13].isnan().all()) and bool(r.entropy[11:13].isnan().all()) and bool(r.entropy[13:].isfinite().all())


def test_tensors_of_another_device_than_the_current_one_are_refused(cuda, monkeypatch):
    """Launches go to the current device: with another one current, every call is refused before anything is launched."""
    x, w = rand(60, (4, 64)), rand(61, (64,))
    target = torch.zeros(4, dtype=torch.int64, device="cuda")
    _, h, rstd = ops.rms_norm(x, w)
    r = ops.log_probs(x, target)
    plan = ops.AdamW([w])
    torch.cuda.synchronize()
    before = w.clone()
    with monkeypatch.context() as m:
        m.setattr(ops, "_current_device", lambda: 1)
        m.setattr(torch.cuda, "current_device", lambda: 1)
        for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_e4m3(x, w), lambda: ops.rms_norm_backward(x, h, w, rstd),
                     lambda: ops.log_probs(x, target), lambda: ops.log_probs_backward(x, target, r.stats, rstd),
                     lambda: ops.AdamW([w]), lambda: plan.step([w.clone()], rate=1.0, t=1)):
            with pytest.raises((ValueError, RuntimeError), match="device"):
                call()
    assert torch.equal(w, before)
