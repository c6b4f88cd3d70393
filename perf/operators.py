"""The operators at the tail of a training step and at a classifier's answer, as cases to time and to check.

Three operators: the root-mean-square norm with the residual's addition (forward, 8-bit output with scales, backward),
log probabilities of given classes with entropy and top alternatives (and their gradient), and an AdamW step over many
tensors (states in 32 or 8 bits).  ``run`` computes a case in elementary torch operations where ``own`` is false and
through ``pixienn_b200.ops`` where it is true; ``exact`` computes it again from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0                    # largest finite value of the 8-bit type
TINY = 2.0 ** -126                  # smallest normal float32: no scale is smaller
BLOCK = 256                         # elements that share one scale of an 8-bit optimiser state
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of a served model: norm and quantisation in front of the next product, latency counts
        dict(name="norm_e4m3_token", op="norm", rows=1, channels=4096, type="bf16", residual=True, group=0, e4m3=True, pad=0),
        # a training step's forward pass over a batch of long sequences
        dict(name="norm_batch", op="norm", rows=16384, channels=4096, type="bf16", residual=True, group=0, e4m3=False, pad=0),
        # a prompt of odd length in front of an 8-bit product, a scale for every 128 channels, a slice of a wider buffer
        dict(name="norm_e4m3_groups", op="norm", rows=2049, channels=5120, type="f16", residual=True, group=128, e4m3=True, pad=128),
        # the training step's way back
        dict(name="norm_back", op="norm_back", rows=8192, channels=2048, type="bf16", residual=True, pad=0),
        # the same in 32 bits with nothing aligned: the features of a small classifier
        dict(name="norm_back_odd", op="norm_back", rows=333, channels=1023, type="f32", residual=False, pad=0),
        # one token's answer out of a large vocabulary, with alternatives
        dict(name="probs_token", op="probs", rows=1, classes=131072, type="f32", top=20, temperature=0.7, masked=0.0, unused=0.0, pad=0),
        # a decoding batch, some classes masked by a grammar
        dict(name="probs_batch", op="probs", rows=64, classes=32000, type="f16", top=8, temperature=1.0, masked=0.25, unused=0.0, pad=0),
        # scoring prompts: an odd vocabulary, padded rows without a target
        dict(name="probs_score", op="probs", rows=4095, classes=50003, type="bf16", top=0, temperature=1.0, masked=0.0, unused=0.1, pad=0),
        # a policy's training step: log probabilities, entropy and the gradient of both
        dict(name="probs_train", op="probs_train", rows=4096, classes=32768, type="bf16", temperature=1.0, masked=0.0, unused=0.05, entropy=True, pad=0),
        # an image classifier's training step (1000 classes, 64 images, 32 bits)
        dict(name="probs_train_images", op="probs_train", rows=64, classes=1000, type="f32", temperature=1.0, masked=0.0, unused=0.0, entropy=False, pad=0),
        # the detector of this repository's benchmark: 222 tensors from 32 to 4.7 million elements, all in 32 bits
        dict(name="adamw_detector", op="adamw", shapes="detector", tensors=0, most=0, shape_seed=0, param="f32", grad="f32", bits=32, master=False),
        # 16-bit parameters with a 32-bit copy, states in 8 bits
        dict(name="adamw_8bit", op="adamw", shapes="spread", tensors=120, most=8388608, shape_seed=7, param="bf16", grad="bf16", bits=8, master=True),
    ]


def _between(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_back", "probs", "probs", "probs_train", "adamw", "adamw"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op in ("norm", "norm_back"):
        channels = _between(rng, 1, 16384)
        if rng.random() < 0.5:
            channels = max(64, channels // 64 * 64)
        rows = _between(rng, 1, max(1, min(65536, (1 << 25) // channels)))
        pad = rng.choice([0, 0, 1, 64])
        case = dict(op=op, rows=rows, channels=channels, type=kind, residual=rng.random() < 0.7, pad=pad)
        if op == "norm":
            case["e4m3"] = rng.random() < 0.5
            case["group"] = rng.choice([0, 32, 64, 128]) if case["e4m3"] else 0
        return case
    if op in ("probs", "probs_train"):
        classes = _between(rng, 2, 262144)
        rows = _between(rng, 1, max(1, min(16384, (1 << 26) // classes)))
        case = dict(op=op, rows=rows, classes=classes, type=kind, temperature=rng.choice([1.0, 1.0, 0.7, 1.5]),
                    masked=rng.choice([0.0, 0.0, 0.3]), unused=rng.choice([0.0, 0.0, 0.2]), pad=rng.choice([0, 0, 1, 8]))
        if op == "probs":
            case["top"] = rng.choice([0, 1, 5, 20, 32])
            if case["top"]:
                case["top"], case["rows"] = min(case["top"], classes), min(rows, max(1, (1 << 24) // classes))
        else:
            case["entropy"] = rng.random() < 0.5
        return case
    bits = rng.choice([8, 32])
    master = kind != "f32" and rng.random() < 0.6
    return dict(op="adamw", shapes="spread", tensors=_between(rng, 1, 200), most=_between(rng, 16, 4194304),
                shape_seed=rng.randrange(1 << 20), param=kind, grad=rng.choice([kind, "f32"]), bits=bits, master=master)


def _sizes(case):
    """Elements of every tensor of an optimiser's case."""
    if case["shapes"] == "detector":
        sizes = []

        def conv(cin, cout, kernel, norm=True):
            sizes.extend([cin * cout * kernel * kernel] + [cout] * (2 if norm else 1))

        conv(3, 32, 3)
        c = 32
        for blocks in (1, 2, 8, 8, 4):                                  # the residual stages of the backbone
            conv(c, 2 * c, 3)
            c *= 2
            for _ in range(blocks):
                conv(c, c // 2, 1)
                conv(c // 2, c, 3)
        cin = c
        for width, skip in ((512, 512), (256, 256), (128, 0)):          # the three heads
            for k in range(3):
                conv(cin if k == 0 else 2 * width, width, 1)
                conv(width, 2 * width, 3)
            conv(2 * width, 255, 1, norm=False)
            if skip:
                conv(width, width // 2, 1)
                cin = width // 2 + skip
        return sizes
    rng = random.Random(case["shape_seed"])
    return [_between(rng, 1, case["most"]) if k else case["most"] for k in range(case["tensors"])]


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, kind, scale=1.0, pad=0):
    """Normal values in a buffer that is `pad` columns wider than the tensor it holds."""
    wide = torch.randn(*shape[:-1], shape[-1] + pad, device="cuda", generator=g).mul_(scale).to(TYPES[kind])
    return wide[..., :shape[-1]]


def _flat(sizes, unit):
    """Offsets of tensors of these sizes in one buffer, each at a multiple of `unit`, and the buffer's length."""
    at, offsets = 0, []
    for n in sizes:
        offsets.append(at)
        at += -(-n // unit) * unit
    return offsets, at


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("norm", "norm_back"):
        n, c = case["rows"], case["channels"]
        s["x"] = _normal(g, (n, c), case["type"], 1.0, case["pad"])
        s["weight"] = torch.rand(c, device="cuda", generator=g).add_(0.5)
        if op == "norm":
            s["residual"] = _normal(g, (n, c), case["type"], 2.0, case["pad"]) if case["residual"] else None
        else:
            s["dy"] = _normal(g, (n, c), case["type"], 0.1, case["pad"])
            s["dresidual"] = _normal(g, (n, c), case["type"], 0.1, case["pad"]) if case["residual"] else None
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + 1e-6)
    elif op in ("probs", "probs_train"):
        n, v = case["rows"], case["classes"]
        x = _normal(g, (n, v), case["type"], 2.5, case["pad"])
        if case["masked"]:                                              # one mask for the batch, as a grammar state gives it
            gone = torch.rand(v, device="cuda", generator=g) < case["masked"]
            gone[0] = False
            x[:, gone] = float("-inf")
        target = torch.randint(0, v, (n,), device="cuda", generator=g)
        if case["masked"]:
            target = torch.where(gone[target], torch.zeros_like(target), target)
        if case["unused"]:
            target = torch.where(torch.rand(n, device="cuda", generator=g) < case["unused"], torch.full_like(target, -1), target)
        s.update(x=x, target=target)
        if op == "probs_train":
            s["dlogp"] = torch.randn(n, device="cuda", generator=g).div_(n)
            s["dentropy"] = torch.full((n,), 0.01 / n, device="cuda") if case["entropy"] else None
    else:
        sizes = _sizes(case)
        offsets, total = _flat(sizes, BLOCK)
        cut = lambda t, per=1: [t[o // per:o // per + -(-n // per)] for o, n in zip(offsets, sizes)]  # noqa: E731
        p = torch.randn(total, device="cuda", generator=g).mul_(0.05)
        grad = torch.randn(total, device="cuda", generator=g).mul_(0.003)
        m = torch.randn(total, device="cuda", generator=g).mul_(0.001)
        r = torch.rand(total, device="cuda", generator=g).mul_(0.003).add_(0.0005)        # the root of the second moment
        s.update(param=p.to(TYPES[case["param"]]), grad=grad.to(TYPES[case["grad"]]), t=100)
        s["master"] = p if case["master"] else None
        if case["bits"] == 32:
            s.update(m=m, v=r.square_())
        else:
            for name, val in (("m", m), ("v", r)):
                blocks = val.view(-1, BLOCK)
                scale = blocks.abs().amax(1).div_(E4M3_MAX).clamp_(min=TINY)
                s[name] = blocks.div_(scale[:, None]).to(torch.float8_e4m3fn).view(-1)
                s[name + "_scale"] = scale
        s["parts"] = {k: cut(s[k], BLOCK if k.endswith("scale") else 1)
                      for k in ("param", "grad", "master", "m", "v", "m_scale", "v_scale") if s.get(k) is not None}
        if own:
            from pixienn_b200 import ops
            q = s["parts"]
            s["plan"] = ops.AdamW(q["param"], state_bits=case["bits"], m=q["m"], v=q["v"], m_scale=q.get("m_scale"),
                                  v_scale=q.get("v_scale"), master=q.get("master"))
    return s


RATE, BETA1, BETA2, EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.01


# ------------------------------------------------------------------------------------------------ plain forms
def _norm_plain(s):
    case, x = s["case"], s["x"]
    if s["residual"] is not None:
        h = (x.float() + s["residual"].float()).to(x.dtype)
    else:
        h = x
    f = h.float()
    rstd = torch.rsqrt(f.square().mean(1) + 1e-6)
    y = f * rstd[:, None] * s["weight"]
    out = {"rstd": rstd}
    if s["residual"] is not None:
        out["h"] = h
    if not case["e4m3"]:
        out["y"] = y.to(x.dtype)
        return out
    n, c = y.shape
    group = case["group"] or c
    groups = -(-c // group)
    wide = torch.zeros(n, groups * group, device=y.device)
    wide[:, :c] = y
    wide = wide.view(n, groups, group)
    scale = (wide.abs().amax(2) / E4M3_MAX).clamp(min=TINY)
    out["q"] = (wide / scale[:, :, None]).view(n, -1)[:, :c].contiguous().to(torch.float8_e4m3fn)
    out["scale"] = scale
    return out


def _norm_back_plain(s):
    h, dy = s["x"].float(), s["dy"].float()
    rstd = s["rstd"][:, None]
    u = dy * s["weight"]
    dx = rstd * (u - h * rstd.square() * (u * h).mean(1, keepdim=True))
    if s["dresidual"] is not None:
        dx = dx + s["dresidual"].float()
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * h * rstd).sum(0)}


def _distances(x, temperature):
    """(x - max x) / T, with rows that are -inf throughout taken from 0."""
    f = x.float()
    m = f.amax(1, keepdim=True)
    return (f - torch.where(m == float("-inf"), torch.zeros_like(m), m)) / temperature


def _probs_plain(s, top):
    target, x = s["target"], s["x"]
    d = _distances(x, s["case"]["temperature"])
    e = d.exp()
    total = e.sum(1)
    logs = total.log()
    used, some = target >= 0, total > 0
    at = d.gather(1, target.clamp(min=0)[:, None])[:, 0]
    zero = torch.zeros_like(logs)
    logp = torch.where(used, torch.where(some, at - logs, at), zero)
    spread = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1) / total
    entropy = torch.where(used & some, logs - spread, zero)
    out = {"logp": logp, "entropy": entropy}
    if top:
        value, index = x.sort(dim=1, descending=True, stable=True)
        index = index[:, :top]
        best = d.gather(1, index)
        best = torch.where(some[:, None], best - logs[:, None], best)
        out["top_logp"] = torch.where(used[:, None], best, torch.zeros_like(best))
        out["top_index"] = torch.where(used[:, None], index, torch.full_like(index, -1)).to(torch.int32)
    return out, d, e, total, logs


def _probs_train_plain(s):
    out, d, e, total, logs = _probs_plain(s, 0)
    target, t = s["target"], s["case"]["temperature"]
    used = ((target >= 0) & (total > 0))[:, None]
    p = e / total[:, None]
    dx = -p * s["dlogp"][:, None]
    if s["dentropy"] is not None:
        dx = dx - s["dentropy"][:, None] * torch.where(p > 0, p * (d - logs[:, None] + out["entropy"][:, None]), torch.zeros_like(p))
    rows = torch.arange(len(target), device=target.device)
    dx[rows, target.clamp(min=0)] += s["dlogp"]
    out["dx"] = torch.where(used, dx / t, torch.zeros_like(dx)).to(s["x"].dtype)
    return out


def _wide(code, scale):
    n = code.numel()
    return code.float() * scale.repeat_interleave(BLOCK)[:n]


def _narrow(val, code, scale, floor):
    """Writes `val` as 8-bit codes with a scale for each block; `floor`: values above zero keep a code above zero."""
    n, blocks = val.numel(), scale.numel()
    wide = torch.zeros(blocks * BLOCK, device=val.device)
    wide[:n] = val
    wide = wide.view(blocks, BLOCK)
    scale.copy_((wide.abs().amax(1) / E4M3_MAX).clamp(min=TINY))
    q = (wide / scale[:, None]).view(-1)[:n]
    if floor:
        q = torch.where(val > 0, q.clamp(min=2.0 ** -9), q)
    code.copy_(q.to(torch.float8_e4m3fn))


def _adamw_plain(s):
    q, small = s["parts"], s["case"]["bits"] == 8
    s["t"] += 1
    c1, c2 = 1 - BETA1 ** s["t"], 1 - BETA2 ** s["t"]
    for k, p in enumerate(q["param"]):
        g = q["grad"][k].float()
        m = _wide(q["m"][k], q["m_scale"][k]) if small else q["m"][k]
        v = _wide(q["v"][k], q["v_scale"][k]).square() if small else q["v"][k]
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        w = q["master"][k] if s["master"] is not None else p.float()
        w = w - RATE * ((m / c1) / ((v / c2).sqrt() + EPS) + DECAY * w)
        if s["master"] is not None:
            q["master"][k].copy_(w)
        p.copy_(w)
        if small:
            _narrow(m, q["m"][k], q["m_scale"][k], False)
            _narrow(v.sqrt(), q["v"][k], q["v_scale"][k], True)
        else:
            q["m"][k].copy_(m)
            q["v"][k].copy_(v)
    return _states(s)


def _states(s):
    return {k: s[k] for k in ("param", "master", "m", "v", "m_scale", "v_scale") if s.get(k) is not None}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    if op == "norm":
        return _norm_plain(state)
    if op == "norm_back":
        return _norm_back_plain(state)
    if op == "probs":
        return _probs_plain(state, state["case"]["top"])[0]
    if op == "probs_train":
        return _probs_train_plain(state)
    return _adamw_plain(state)


def _run_own(op, s):
    from pixienn_b200 import ops
    case = s["case"]
    if op == "norm":
        if case["e4m3"]:
            q, scale, h, rstd = ops.rms_norm_e4m3(s["x"], s["weight"], residual=s["residual"], eps=1e-6, group=case["group"])
            out = {"q": q, "scale": scale, "rstd": rstd}
        else:
            y, h, rstd = ops.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=1e-6)
            out = {"y": y, "rstd": rstd}
        if s["residual"] is not None:
            out["h"] = h
        return out
    if op == "norm_back":
        dx, dweight = ops.rms_norm_backward(s["dy"], s["x"], s["weight"], s["rstd"], dresidual=s["dresidual"])
        return {"dx": dx, "dweight": dweight}
    if op in ("probs", "probs_train"):
        r = ops.log_probs(s["x"], s["target"], top=case.get("top", 0), temperature=case["temperature"])
        out = {"logp": r.logp, "entropy": r.entropy}
        if case.get("top", 0):
            out.update(top_logp=r.top_logp, top_index=r.top_index)
        if op == "probs_train":
            out["dx"] = ops.log_probs_backward(s["x"], s["target"], r.stats, s["dlogp"], dentropy=s["dentropy"], temperature=case["temperature"])
        return out
    s["t"] += 1
    s["plan"].step(s["parts"]["grad"], rate=RATE, t=s["t"], beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY)
    return _states(s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op in ("norm", "norm_back"):
        n, c, b = case["rows"], case["channels"], BYTES[case["type"]]
        if op == "norm_back":
            return {"bytes": n * c * b * (4 if case["residual"] else 3) + 4 * n + 8 * c, "flops": 11 * n * c}
        moved = n * c * b * (3 if case["residual"] else 1) + 4 * n + 4 * c
        if case["e4m3"]:
            return {"bytes": moved + n * c + 4 * n * -(-c // (case["group"] or c)), "flops": 9 * n * c}
        return {"bytes": moved + n * c * b, "flops": 6 * n * c}
    if op in ("probs", "probs_train"):
        n, v, b = case["rows"], case["classes"], BYTES[case["type"]]
        read = n * (1 - case["unused"]) * v * b + n * (16 + 8 * case.get("top", 0))
        if op == "probs":
            return {"bytes": read, "flops": 6 * n * v}
        # the gradient needs the row's sums first: its values are read a second time, unused rows are only written
        return {"bytes": 2 * read + n * v * b, "flops": 12 * n * v}
    n = sum(_sizes(case))
    per = BYTES[case["grad"]] + BYTES[case["param"]] + (8 if case["master"] else BYTES[case["param"]])
    per += 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * per, "flops": 16 * n}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _norm_exact(s)
    if op == "norm_back":
        return _norm_back_exact(s)
    if op == "probs":
        return _probs_exact(s, case["top"], False)
    if op == "probs_train":
        return _probs_exact(s, 0, True)
    return _adamw_exact(s)


def _norm_exact(s):
    case, x = s["case"], s["x"].double()
    out = {}
    if s["residual"] is not None:
        x = x + s["residual"].double()
        out["h"] = x
        x = x.to(s["x"].dtype).double()             # the norm is that of the stored sum
    mean = torch.einsum("nc,nc->n", x, x) / x.shape[1]
    out["rstd"] = 1.0 / torch.sqrt(mean + 1e-6)
    y = torch.einsum("nc,n,c->nc", x, out["rstd"], s["weight"].double())
    if not case["e4m3"]:
        return {**out, "y": y}
    group = case["group"] or case["channels"]
    parts = [y[:, k:k + group] for k in range(0, case["channels"], group)]
    scales = [torch.clamp(p.abs().max(dim=1, keepdim=True).values / E4M3_MAX, min=TINY) for p in parts]
    # an 8-bit value's counterpart is what is rounded to it
    return {**out, "q": torch.cat([p / k for p, k in zip(parts, scales)], 1), "scale": torch.cat(scales, 1)}


def _norm_back_exact(s):
    x, dy, w, r = s["x"].double(), s["dy"].double(), s["weight"].double(), s["rstd"].double()
    xhat = x * r[:, None]
    back = torch.einsum("nc,nc,c->n", dy, xhat, w) / x.shape[1]
    dx = (dy * w - xhat * back[:, None]) * r[:, None]
    if s["dresidual"] is not None:
        dx += s["dresidual"].double()
    return {"dx": dx, "dweight": torch.einsum("nc,nc->c", dy, xhat)}


def _probs_exact(s, top, train):
    case, target = s["case"], s["target"]
    n, v = case["rows"], case["classes"]
    out = {"logp": torch.zeros(n, dtype=torch.float64, device="cuda"), "entropy": torch.zeros(n, dtype=torch.float64, device="cuda")}
    if top:
        out["top_logp"] = torch.zeros(n, top, dtype=torch.float64, device="cuda")
        out["top_index"] = torch.full((n, top), -1, dtype=torch.int32, device="cuda")
    if train:
        out["dx"] = torch.zeros(n, v, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // v)
    for a in range(0, n, step):
        rows = a + torch.nonzero(target[a:a + step] >= 0)[:, 0]
        if not len(rows):
            continue
        z = s["x"][rows].double() / case["temperature"]
        lse = torch.logsumexp(z, 1)
        lp = z - lse[:, None]
        p = torch.exp(lp)
        plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
        h = -plogp.sum(1)
        t = target[rows]
        out["logp"][rows] = lp[torch.arange(len(rows), device="cuda"), t]
        out["entropy"][rows] = h
        if top:
            order = torch.argsort(-s["x"][rows].double(), dim=1, stable=True)[:, :top]
            out["top_index"][rows] = order.to(torch.int32)
            out["top_logp"][rows] = torch.gather(lp, 1, order)
        if train:
            dx = -p * s["dlogp"][rows].double()[:, None]
            if s["dentropy"] is not None:
                dx -= (plogp + p * h[:, None]) * s["dentropy"][rows].double()[:, None]
            dx.scatter_add_(1, t[:, None], s["dlogp"][rows].double()[:, None])
            out["dx"][rows] = dx / case["temperature"]
    return out


def _adamw_exact(s):
    """One step on the whole buffers at once: the tensors lie in them at multiples of a block, and what lies between two
    tensors is left as it is."""
    case, t = s["case"], s["t"] + 1
    sizes = _sizes(case)
    offsets, total = _flat(sizes, BLOCK)
    inside = torch.zeros(total + 1, dtype=torch.int32, device="cuda")
    inside.index_add_(0, torch.tensor(offsets, device="cuda"), torch.ones(len(sizes), dtype=torch.int32, device="cuda"))
    inside.index_add_(0, torch.tensor([o + n for o, n in zip(offsets, sizes)], device="cuda"), torch.full((len(sizes),), -1, dtype=torch.int32, device="cuda"))
    inside = inside.cumsum(0)[:total] > 0
    g = s["grad"].double()
    old = (s["master"] if s["master"] is not None else s["param"]).double()
    if case["bits"] == 8:
        m0 = (s["m"].double().view(-1, BLOCK) * s["m_scale"].double()[:, None]).view(-1)
        r0 = (s["v"].double().view(-1, BLOCK) * s["v_scale"].double()[:, None]).view(-1)
        v0 = r0 * r0
    else:
        m0, v0 = s["m"].double(), s["v"].double()
    m = m0 + (1 - BETA1) * (g - m0)
    v = v0 + (1 - BETA2) * (g * g - v0)
    root = torch.sqrt(v)
    step = m / (1 - BETA1 ** t) / (root / math.sqrt(1 - BETA2 ** t) + EPS)
    w = old * (1 - RATE * DECAY) - RATE * step
    out = {"param": torch.where(inside, w, s["param"].double())}
    if s["master"] is not None:
        out["master"] = torch.where(inside, w, old)
    if case["bits"] == 32:
        return {**out, "m": torch.where(inside, m, m0), "v": torch.where(inside, v, v0)}
    for name, val in (("m", m), ("v", root)):
        blocks = torch.where(inside, val, torch.zeros_like(val)).view(-1, BLOCK)
        scale = torch.clamp(blocks.abs().amax(1) / E4M3_MAX, min=TINY)
        # an 8-bit value's counterpart is what is rounded to it
        out[name] = torch.where(inside, (blocks / scale[:, None]).view(-1), s[name].double())
        out[name + "_scale"] = scale
    return out
