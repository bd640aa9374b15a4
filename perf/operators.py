"""Cases and plain forms of the compact optimizer state: the AdamW step with
8-bit moments, the NorMuon momentum pass with an 8-bit momentum, and the
conversions between 8-bit and wide states.

The 8-bit form of a state: blocks of 128 consecutive elements of the flattened
tensor, each with one fp32 scale s.
  signed (first moments): s = max |x|,      code q = sgn(x) floor(127 sqrt(|x| / s) + u),  value s q |q| / 127^2
  root (second moments):  s = max sqrt(x),  code q = floor(255 sqrt(sqrt(x) / s) + u), at least 1 where x > 0,
                                            value (s (q / 255)^2)^2
  pair (master weights):  bf16 weight p = bf16(w) and remainder bf16(w - p), value p + remainder
u is 1/2 (nearest) in a conversion. In a step it runs evenly over [0, 1) from
step to step, so that a change smaller than a code step is kept on average:
with h = 2654435769 i + 1779033703 t (+ 2^31 for signed) modulo 2^32 for element
i in step t, u = floor(h / 2^9) / 2^23. A block that holds a value that is not
finite has the scale NaN; one that holds only zeros has the scale 0.
"""
import ctypes
import math
import os
import sys

import torch

own = False

BLOCK = 128
PART = 16384  # elements of a matrix behind one partial sum of squares of the momentum pass


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # the recipe's gains, gates and scalars in one call: latency
        {"name": "adamw gains", "op": "adamw", "dtype": "bf16", "shapes": "1024,1024,1024,1024,8,8x12,1,12,1024,8",
         "master": True, "ema": False, "wd": 0.0, "cautious": False, "beta2": 0.95},
        # a small fp32 model with odd shapes, cautious decay and an EMA
        {"name": "adamw odd fp32", "op": "adamw", "dtype": "fp32", "shapes": "333x77,4099,5x64x33,1024x128",
         "master": False, "ema": True, "wd": 0.1, "cautious": True, "beta2": 0.999},
        # one vocabulary table of the recipe, bf16 weights alone
        {"name": "adamw table", "op": "adamw", "dtype": "bf16", "shapes": "32768x1024",
         "master": False, "ema": False, "wd": 0.01, "cautious": False, "beta2": 0.95},
        # every vocabulary table of the recipe: master weights and EMA
        {"name": "adamw tables ema", "op": "adamw", "dtype": "bf16", "shapes": "32768x1024,32768x1024,5x32768x1024",
         "master": True, "ema": True, "wd": 0.0, "cautious": False, "beta2": 0.95},
        # the matrices of a three-layer model of width 128
        {"name": "momentum small", "op": "momentum", "dtype": "bf16", "shapes": "3x128x128,3x4x128,3x384x128,3x128x384",
         "nesterov": True},
        # matrices whose rows end inside a block and inside a vector
        {"name": "momentum odd fp32", "op": "momentum", "dtype": "fp32", "shapes": "2x333x77,1x1x5,3x257x129",
         "nesterov": False},
        # the recipe's matrices of 14 layers, one call
        {"name": "momentum 14 layers", "op": "momentum", "dtype": "bf16",
         "shapes": "14x1024x1024,14x8x1024,14x5632x1024,14x1024x5632", "nesterov": True},
        # the state of a small model written in 8 bits when a 32-bit checkpoint is loaded
        {"name": "encode small", "op": "encode", "dtype": "fp32", "shapes": "128x384,333x77,129,1,1000"},
        # the moments of a vocabulary table, bf16
        {"name": "encode table", "op": "encode", "dtype": "bf16", "shapes": "32768x1024"},
        # the state of a small model read back for a checkpoint
        {"name": "decode small", "op": "decode", "dtype": "bf16", "shapes": "128x384,333x77,129,1,1000"},
        # a vocabulary table's moments and master weights read back in 32 bits
        {"name": "decode table", "op": "decode", "dtype": "fp32", "shapes": "32768x1024"},
    ]


def _size(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["adamw", "adamw", "momentum", "encode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "momentum":
        batches = []
        for _ in range(rng.randint(1, 4)):
            r, c = _size(rng, 1, 6000), _size(rng, 1, 6000)
            batches.append("%dx%dx%d" % (min(rng.randint(1, 14), max(1, 40_000_000 // (r * c))), r, c))
        return {"op": op, "dtype": dtype, "shapes": ",".join(batches), "nesterov": rng.random() < 0.7}
    tensors = []
    for _ in range(rng.randint(1, 6)):
        n = _size(rng, 1, 20_000_000)
        cols = _size(rng, 1, 2000)
        tensors.append("%dx%d" % (max(1, n // cols), cols) if rng.random() < 0.6 else "%d" % n)
    case = {"op": op, "dtype": dtype, "shapes": ",".join(tensors)}
    if op == "adamw":
        wd = rng.choice([0.0, 0.01, 0.1])
        case |= {"master": dtype == "bf16" and rng.random() < 0.6, "ema": rng.random() < 0.5, "wd": wd,
                 "cautious": rng.random() < 0.5, "beta2": rng.choice([0.95, 0.99, 0.999])}
    return case


def _shapes(case):
    return [tuple(int(d) for d in s.split("x")) for s in case["shapes"].split(",")]


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


LR, BETA1, EPS, DECAY, MOMENTUM, STEP = 1.2e-2, 0.9, 1e-8, 0.999, 0.95, 20


def work(case):
    shapes = _shapes(case)
    n = sum(math.prod(s) for s in shapes)
    t = 2 if case["dtype"] == "bf16" else 4
    blocks = 4.0 * n / BLOCK  # bytes of one state's scales
    if case["op"] == "adamw":
        # weight in and out, gradient, two codes in and out with their scales, the moments as bf16 values;
        # remainder in and out and the fp32 master weight; EMA in and out
        per = 3 * t + 4 + 4 + (8 if case["master"] else 0) + (8 if case["ema"] else 0)
        return {"bytes": per * n + 4 * blocks, "flops": 40 * n}
    if case["op"] == "momentum":
        # gradient, code in and out with its scale, u, the momentum as bf16 values
        return {"bytes": (t + 2 + 2 + 2) * n + 2 * blocks, "flops": 20 * n}
    if case["op"] == "encode":
        # two states read and written, and the values that the codes stand for, bf16
        return {"bytes": (2 * t + 2 + 4) * n + 2 * blocks, "flops": 20 * n}
    # two codes and a bf16 pair read, three values written
    return {"bytes": (2 + 4 + 2 * t + 4) * n + 2 * blocks, "flops": 8 * n}


# ----------------------------------------------------------------- inputs ---
def _like(shape, gen, std):
    """Values as gradients have them: 5 % of the rows ten times as large, and 10 % of the rows not touched at all."""
    x = torch.randn(shape, generator=gen, device="cuda") * std
    if len(shape) > 1:
        rows = x.view(-1, shape[-1])
        u = torch.rand(rows.shape[0], 1, generator=gen, device="cuda")
        rows *= torch.where(u < 0.05, 10.0, torch.where(u > 0.9, 0.0, 1.0))
    return x


def _inputs(case, seed):
    """Seeded inputs of one case, without the framework's objects."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, s = _dtype(case), {"case": case, "items": []}
    for shape in _shapes(case):
        one = {}
        if case["op"] == "momentum":
            one["g"] = _like(shape, gen, 1e-3).to(dt)
            kept = [_write_signed(x) for x in _like(shape, gen, 5e-4)]
            one["m"] = torch.stack([q for q, _ in kept])
            one["ms"] = torch.stack([sc for _, sc in kept])
        else:
            seen = _like(shape, gen, 1e-3)
            m = 0.5 * seen + 0.3 * seen.roll(1)
            v = seen.square() * (0.5 + torch.rand(shape, generator=gen, device="cuda"))
            if case["op"] == "encode":
                one["m"], one["v"] = m.to(dt), v.to(dt)
            else:
                (one["m"], one["ms"]), (one["v"], one["vs"]) = _write_signed(m), _write_root(v)
                w = torch.randn(shape, generator=gen, device="cuda") * 0.02
                pair = case["op"] == "decode" or case["master"]
                one["p"] = w.to(torch.bfloat16 if pair else dt)
                one["rem"] = (w - one["p"].float()).to(torch.bfloat16) if pair else None
                one["g"] = (seen + torch.randn(shape, generator=gen, device="cuda") * 2e-4 * (seen != 0)).to(dt)
                one["ema"] = w + torch.randn(shape, generator=gen, device="cuda") * 1e-3 if case.get("ema") else None
        s["items"].append(one)
    s["t"] = STEP
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _handles(case, s)
    return s


# ------------------------------------------------------------- plain form ---
def _blocks(x):
    flat = x.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def _dither(b, t, phase):
    if t is None:
        return 0.5
    i = torch.arange(b.numel(), device=b.device).view(b.shape)
    return ((i * 2654435769 + t * 1779033703 + phase) % 2 ** 32 // 2 ** 9).double() / 2 ** 23


def _code(x, s, levels, u):
    """floor(levels sqrt(x / s) + u): in 64 bits, so that the side of a border does not hang on a rounding."""
    y = levels * (x.double() / torch.where(s > 0, s, 1.0).double()[:, None]).sqrt()
    return torch.where((s > 0)[:, None], (y + u).floor().clamp(max=levels), 0.0)


def _write_signed(x, t=None):
    b = _blocks(x.float())
    s = b.abs().amax(1)
    s = torch.where(s.isfinite(), torch.where(s >= 2.0 ** -126, s, 0.0), math.nan)
    q = _code(b.abs(), s, 127, _dither(b, t, 2 ** 31)) * b.sign()
    return q.to(torch.int8).view(-1)[: x.numel()].view(x.shape), s


def _write_root(x, t=None):
    b = _blocks(x.float())
    s = b.amax(1).sqrt()
    s = torch.where(s.isfinite(), s, math.nan)
    q = torch.maximum(_code(b.sqrt(), s, 255, _dither(b, t, 0)), ((b > 0) & (s > 0)[:, None]).double())
    return q.to(torch.uint8).view(-1)[: x.numel()].view(x.shape), s


def _read_signed(q, s):
    f = _blocks(q).float()
    return (f * f.abs() * (1 / 16129) * s[:, None]).view(-1)[: q.numel()].view(q.shape)


def _read_root(q, s):
    f = _blocks(q).float()
    return (f * f * (1 / 65025) * s[:, None]).square().view(-1)[: q.numel()].view(q.shape)


def _plain_adamw(case, one, t):
    b2, wd = case["beta2"], case["wd"]
    g = one["g"].float()
    m = BETA1 * _read_signed(one["m"], one["ms"]) + (1 - BETA1) * g
    v = b2 * _read_root(one["v"], one["vs"]) + (1 - b2) * (g * g)
    w = one["p"].float() if one["rem"] is None else one["p"].float() + one["rem"].float()
    if wd and case["cautious"]:
        w = w * (1 - LR * wd * (m * w > 0).float())
    elif wd:
        w = w - LR * wd * w
    w = w - LR / (1 - BETA1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + EPS)
    p = one["p"].copy_(w)
    one["m"], one["ms"] = _write_signed(m, t)
    one["v"], one["vs"] = _write_root(v, t)
    out = {"p": p, "exp_avg": _read_signed(one["m"], one["ms"]).bfloat16(),
           "exp_avg_sq": _read_root(one["v"], one["vs"]).bfloat16()}
    if one["rem"] is not None:
        one["rem"].copy_(w - p.float())
        out["master"] = p.float() + one["rem"].float()
    if one["ema"] is not None:
        out["ema"] = one["ema"].add_((1 - DECAY) * (p.float() - one["ema"]))
    return out


def _plain_momentum(case, one, t):
    shape = one["g"].shape
    many = [_plain_matrix(case, one["g"][i].float(), one["m"][i], one["ms"][i], t) for i in range(shape[0])]
    u, sq, m, ms, val = (torch.stack(x) for x in zip(*many))
    one["m"], one["ms"] = m, ms
    return {"u": u, "squares": sq, "momentum": val}


def _plain_matrix(case, g, q, s, t):
    m, s = _write_signed(MOMENTUM * _read_signed(q, s) + (1 - MOMENTUM) * g, t)
    val = _read_signed(m, s)
    u = (MOMENTUM * val + (1 - MOMENTUM) * g if case["nesterov"] else val).bfloat16()
    sq = u.float().square().view(-1)
    sq = torch.nn.functional.pad(sq, (0, -sq.numel() % PART)).view(-1, PART).sum(1)
    return u, sq, m, s, val.bfloat16()


def _plain_encode(one):
    (m, ms), (v, vs) = _write_signed(one["m"]), _write_root(one["v"])
    return {"exp_avg": _read_signed(m, ms).bfloat16(), "exp_avg_scale": ms,
            "exp_avg_sq": _read_root(v, vs).bfloat16(), "exp_avg_sq_scale": vs}


def _plain_decode(case, one):
    dt = _dtype(case)
    return {"exp_avg": _read_signed(one["m"], one["ms"]).to(dt), "exp_avg_sq": _read_root(one["v"], one["vs"]).to(dt),
            "master": one["p"].float() + one["rem"].float()}


def run(s):
    if own:
        return _own(s)
    case, s["t"] = s["case"], s["t"] + 1
    if case["op"] == "adamw":
        return [_plain_adamw(case, one, s["t"]) for one in s["items"]]
    if case["op"] == "momentum":
        return [_plain_momentum(case, one, s["t"]) for one in s["items"]]
    if case["op"] == "encode":
        return [_plain_encode(one) for one in s["items"]]
    return [_plain_decode(case, one) for one in s["items"]]


# ------------------------------------------------------- the framework's ---
def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cs336-a1-sol_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import sol_b200
    return sol_b200


def _handles(case, s):
    """What a training program keeps: the optimizer with its state, the EMA, the launch descriptors."""
    sol = _package()
    if case["op"] == "adamw":
        ps = [torch.nn.Parameter(one["p"]) for one in s["items"]]
        s["opt"] = opt = sol.AdamW([{"params": ps, "lr": LR, "weight_decay": case["wd"]}], betas=(BETA1, case["beta2"]),
                                   eps=EPS, master="bf16_mt" if case["master"] else "none", state_dtype=torch.int8,
                                   min_8bit_numel=0, cautious_wd=case["cautious"])
        state = {}
        for i, (p, one) in enumerate(zip(ps, s["items"])):
            p.grad = one["g"]
            state[i] = {"step": torch.tensor(float(STEP), device="cuda"), "exp_avg": one["m"], "exp_avg_scale": one["ms"],
                        "exp_avg_sq": one["v"], "exp_avg_sq_scale": one["vs"]}
            if one["rem"] is not None:
                state[i]["mant_rem"] = one["rem"]
        opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
        s["params"], s["ema"] = ps, None
        if case["ema"]:
            s["ema"] = sol.EmaWeights(torch.nn.ParameterList(ps), DECAY)
            s["ema"].update()  # from here on the step keeps the average
            for shadow, one in zip(s["ema"].shadow, s["items"]):
                shadow.copy_(one["ema"])
    elif case["op"] == "momentum":
        from sol_b200 import _lib
        lib, keep = _lib.load(), []
        arr, scales, steps = (_lib.NormuonBatch * len(s["items"]))(), [], []
        for i, one in enumerate(s["items"]):
            S, r, c = one["g"].shape
            one["u"] = torch.empty(S, r, c, dtype=torch.bfloat16, device="cuda")
            one["val"] = torch.empty_like(one["u"])
            one["sq"] = torch.empty(S, lib.b2o_normuon_front_parts(r * c), device="cuda")
            grads = _lib.ptr_array([x.data_ptr() for x in one["g"]])
            bufs = _lib.ptr_array([x.data_ptr() for x in one["m"]])
            sc = _lib.ptr_array([x.data_ptr() for x in one["ms"]])
            keep += [grads, bufs, sc]
            scales.append(_lib.addr(sc))
            steps.append((ctypes.c_uint32 * S)())
            arr[i] = _lib.NormuonBatch(S=S, r=r, c=c, grads=_lib.addr(grads), bufs=_lib.addr(bufs),
                                       u=one["u"].data_ptr(), partial=one["sq"].data_ptr())
        s["steps"] = steps
        s["call"] = (arr, _lib.ptr_array(scales), _lib.ptr_array([_lib.addr(x) for x in steps]), len(s["items"]), _lib.dtype_code(_dtype(case)), MOMENTUM,
                     int(case["nesterov"]), None)
        s["keep"] = keep


def _own(s):
    case, items = s["case"], s["items"]
    sol = _package()
    if case["op"] == "adamw":
        s["opt"].step()
        if s["ema"] is not None:
            s["ema"].update()
        out = [{"p": p.data, **x} for p, x in zip(s["params"], s["opt"].expanded_state(s["params"], torch.bfloat16))]
        if s["ema"] is not None:
            for x, shadow in zip(out, s["ema"].shadow):
                x["ema"] = shadow
        return out
    from sol_b200 import state8
    if case["op"] == "momentum":
        from sol_b200 import _lib
        s["t"] += 1
        for x in s["steps"]:
            x[:] = [s["t"]] * len(x)
        _lib.check(_lib.load().b2o_normuon_front8_multi(*s["call"], _lib.stream_ptr()), "normuon_front8")
        state8.decode([(q, sc, "signed") for one in items for q, sc in zip(one["m"], one["ms"])],
                      out=[x for one in items for x in one["val"]])
        return [{"u": one["u"], "squares": one["sq"], "momentum": one["val"]} for one in items]
    if case["op"] == "encode":
        kept = state8.encode([x for one in items for x in ((one["m"], "signed"), (one["v"], "root"))])
        vals = state8.decode([(q, sc, k) for (q, sc), k in zip(kept, ("signed", "root") * len(items))], dtype=torch.bfloat16)
        return [{"exp_avg": vals[i], "exp_avg_scale": kept[i][1], "exp_avg_sq": vals[i + 1], "exp_avg_sq_scale": kept[i + 1][1]}
                for i in range(0, len(kept), 2)]
    dt = _dtype(case)
    vals = state8.decode([x for one in items for x in ((one["m"], one["ms"], "signed"), (one["v"], one["vs"], "root"),
                                                       (one["p"], one["rem"], "pair"))],
                         dtype=[dt, dt, torch.float32] * len(items))
    return [{"exp_avg": vals[i], "exp_avg_sq": vals[i + 1], "master": vals[i + 2]} for i in range(0, len(vals), 3)]


# -------------------------------------------------------- 64-bit results ---
def _coded(x, root, step=None):
    """The value that the 8-bit code of each element stands for, from the definition, in 64 bits."""
    n, levels = x.numel(), 255.0 if root else 127.0
    size = x.abs().sqrt() if root else x.abs()
    rows = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    rows[:n] = size.reshape(-1)
    rows = rows.view(-1, BLOCK)
    top = rows.max(dim=1, keepdim=True).values.float().double()  # scales are kept in 32 bits
    part = torch.full_like(rows, 0.5)
    if step is not None:
        turn = torch.arange(rows.numel(), device=x.device).mul_(0x9E3779B9).add_((0x6A09E667 * step + (0 if root else 1 << 31)) & 0xFFFFFFFF)
        part = ((turn & 0xFFFFFFFF) >> 9).view(rows.shape).double().mul_(2.0 ** -23)
    q = torch.floor(levels * torch.sqrt(torch.nan_to_num(rows / top)) + part).clamp_(max=levels)
    if root:
        q = torch.maximum(q, (rows > 0).double())
    size = (top * (q / levels) ** 2).view(-1)[:n].view(x.shape)
    return (size * size if root else torch.copysign(size, x)), top.view(-1)


def _stands_for(q, scale, root):
    q64 = q.double().reshape(-1)
    y = q64.abs() / (255.0 if root else 127.0)
    y = y * y * scale.double().repeat_interleave(BLOCK)[: q.numel()]
    return (y * y if root else torch.copysign(y, q64)).view(q.shape)


def exact(case, seed):
    out = []
    for one in _inputs(case, seed)["items"]:
        if case["op"] == "adamw":
            b2, t = case["beta2"], STEP + 1
            g = one["g"].double()
            m = _stands_for(one["m"], one["ms"], False).mul_(BETA1).add_(g, alpha=1 - BETA1)
            v = _stands_for(one["v"], one["vs"], True).mul_(b2).addcmul_(g, g, value=1 - b2)
            del g
            w = one["p"].double()
            if one["rem"] is not None:
                w = w + one["rem"].double()
            if case["wd"]:
                shrink = torch.full_like(w, LR * case["wd"])
                if case["cautious"]:
                    shrink[m * w <= 0] = 0
                w = w * (1 - shrink)
            root = (v / (1 - b2 ** t)).sqrt()
            w = w - LR * (m / (1 - BETA1 ** t)) / (root + EPS)
            d = {"p": w, "exp_avg": _coded(m, False, t)[0], "exp_avg_sq": _coded(v, True, t)[0]}
            if one["rem"] is not None:
                d["master"] = w
            if one["ema"] is not None:
                d["ema"] = one["ema"].double() * DECAY + (1 - DECAY) * w.to(_dtype(case)).double()
        elif case["op"] == "momentum":
            d = {"u": [], "squares": [], "momentum": []}
            for g, q, sc in zip(one["g"].double(), one["m"], one["ms"]):
                val = _coded(MOMENTUM * _stands_for(q, sc, False) + (1 - MOMENTUM) * g, False, STEP + 1)[0]
                u = MOMENTUM * val + (1 - MOMENTUM) * g if case["nesterov"] else val
                d["u"].append(u)
                parts = u.to(torch.bfloat16).double().square().flatten().split(PART)
                d["squares"].append(torch.stack([x.sum() for x in parts]))
                d["momentum"].append(val)
            d = {k: torch.stack(x) for k, x in d.items()}
        elif case["op"] == "encode":
            m, ms = _coded(one["m"].double(), False)
            v, vs = _coded(one["v"].double(), True)
            d = {"exp_avg": m, "exp_avg_scale": ms, "exp_avg_sq": v, "exp_avg_sq_scale": vs}
        else:
            d = {"exp_avg": _stands_for(one["m"], one["ms"], False), "exp_avg_sq": _stands_for(one["v"], one["vs"], True),
                 "master": one["p"].double() + one["rem"].double()}
        out.append(d)
    return out
