"""Grouped-head attention over a cache held in 8 bits: what writes the cache, reads it back, takes a decode step on it and attends with a prompt's portion.

A head's key (of one map) and a head's value at a position are whole numbers -127 .. 127 with one scale each: a = largest magnitude, scale = a / 127, number =
value * (127 / a) to the nearest, ties to even.  Keys int8 [kv heads][maps][capacity][dimp]; values int8 [kv heads][capacity / 32][vdimp / 32][16][4][2][8],
column c at position p in [p / 32][c / 32][c % 16][p % 32 / 8][c % 32 / 16][p % 8]; scales f32 [kv heads][maps][capacity] and [kv heads][capacity].
dimp, vdimp: the columns up to a multiple of 32, zero behind the head's own.

A case's "op" names the operator:
  write   n rows of projections from position `first` on: queries out, keys and values into the cache, which come back as the bf16 values they stand for
  read    n positions from `first` on as bf16 or f32
  step    one token at position `first`, the keys ahead of it in the cache: the heads' outputs in f32, and what the cache holds at that position
  prompt  the last n of `first` + n positions attend, all of them in the cache: bf16
"""
import importlib
import math

import torch

own = False

EPS, LAMBDA, OUT_SCALE = 1e-5, 0.4, 0.6


def listed():
    def case(name, op, heads, kv_heads, dim, vdim, first, n, maps=1, rot=0, window=0, f32=False):
        return {"name": name, "op": op, "heads": heads, "kv_heads": kv_heads, "maps": maps, "dim": dim, "vdim": vdim, "rot": rot, "first": first, "n": n, "window": window, "f32": f32}

    return [
        # one token's keys and values written apart from the attention: latency
        case("write 1", "write", 20, 5, 128, 128, 700, 1, rot=64, f32=True),
        # a second portion of a prompt, of differential attention: positions begin inside a tile
        case("write 1531 two maps", "write", 12, 3, 64, 128, 37, 1531, maps=2),
        # a long prompt in one portion
        case("write 16384", "write", 20, 5, 128, 128, 0, 16384, rot=64),
        # a short cache handed to a program that wants f32; heads that are no multiple of 32 columns
        case("read 300 f32", "read", 12, 3, 80, 80, 5, 300, f32=True),
        # a long cache handed over in bf16
        case("read 131072", "read", 32, 8, 128, 128, 0, 131072),
        # a chat's step: latency
        case("step 200", "step", 20, 5, 128, 128, 199, 1, rot=64),
        # a step of differential attention
        case("step 2090 two maps", "step", 12, 3, 64, 128, 2089, 1, maps=2),
        # a step within a window, wide heads in groups of eight
        case("step 30011 window", "step", 16, 2, 256, 256, 30010, 1, rot=128, window=4096),
        # a step behind a very long context: bandwidth
        case("step 131072", "step", 32, 8, 128, 128, 131071, 1, rot=64),
        # a short prompt
        case("prompt 130", "prompt", 12, 3, 128, 128, 0, 130),
        # a question behind a long document, differential attention
        case("prompt 509 of 20520", "prompt", 12, 3, 64, 128, 20011, 509, maps=2),
        # a long prompt in one portion
        case("prompt 8192", "prompt", 20, 5, 128, 128, 0, 8192),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["write", "read", "step", "prompt"])
    kv_heads = rng.choice([1, 2, 3, 5, 6, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    maps = rng.choice([1, 1, 2])
    dim = rng.choice([40, 64, 80, 96, 128] + ([160, 256] if maps == 1 else []))
    vdim = rng.choice([dim, 64, 128]) if maps == 2 else dim
    rot = rng.choice([0, dim // 2, dim])
    f32, window, first, n = False, 0, 0, 1
    if op == "write":
        n, f32 = spread(1, 8192), rng.random() < 0.3
        first = rng.choice([0, rng.randrange(1, 5000)])
    elif op == "read":
        n, f32 = spread(1, 60000), rng.random() < 0.3
        first = rng.randrange(0, 2000)
    elif op == "step":
        first = spread(1, 100000) - 1
        window = rng.choice([0, 0, spread(16, 8192)])
    else:
        n = spread(2, 3000)
        first = rng.choice([0, spread(1, 8000)])
        window = rng.choice([0, 0, 0, spread(16, 4096)])
    return {"op": op, "heads": heads, "kv_heads": kv_heads, "maps": maps, "dim": dim, "vdim": vdim, "rot": rot, "first": first, "n": n, "window": window, "f32": f32}


def up_to(n, step):
    return -(-n // step) * step


def visible(case):
    """(query, key) pairs of an attention case, and the keys that some query sees"""
    first, n, window = case["first"], case["n"], case["window"] or 1 << 40
    if n <= 4096:
        pairs = sum(min(first + i + 1, window) for i in range(n))
    else:
        at = torch.arange(first + 1, first + n + 1, dtype=torch.int64)
        pairs = int(at.clamp(max=min(window, 1 << 40)).sum())
    return pairs, min(first + n, window + n - 1)


def work(case):
    H, G, M, D, V, n = case["heads"], case["kv_heads"], case["maps"], case["dim"], case["vdim"], case["n"]
    t, held, row = 4 if case["f32"] else 2, G * (M * D + V + 4 * M + 4), H * M * D + G * (M * D + V)
    if case["op"] == "write":
        return {"bytes": n * (row * t + H * M * D * t + held + G * (M * D + V) * 2), "flops": 8 * n * row}
    if case["op"] == "read":
        return {"bytes": n * (held + G * (M * D + V) * t), "flops": n * G * (M * D + V)}
    pairs, keys = visible(case)
    flops = 2 * H * M * (D + V) * pairs
    if case["op"] == "step":
        return {"bytes": keys * held + row * 4 + H * V * 4, "flops": flops}
    return {"bytes": keys * held + n * H * (M * D + V) * 2, "flops": flops}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def pack_values(numbers):
    """int8 [kv heads][capacity][vdimp] -> the cache's order"""
    G, C, V = numbers.shape
    return numbers.view(G, C // 32, 4, 8, V // 32, 2, 16).permute(0, 1, 4, 6, 2, 5, 3).contiguous()


def stored(x):
    """vectors along the last axis -> numbers, scales"""
    largest = x.abs().amax(-1)
    live = largest >= 1.5e-36
    scale = torch.where(live, largest / 127, torch.zeros_like(largest))
    factor = torch.where(live, 127 / largest, torch.zeros_like(largest))
    return torch.round(x * factor[..., None]), scale


def prepare(case, seed):
    H, G, M, D, V, first, n = (case[k] for k in ("heads", "kv_heads", "maps", "dim", "vdim", "first", "n"))
    Dp, Vp, half = up_to(D, 32), up_to(V, 32), case["rot"] // 2
    C = up_to(first + n, 128)
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": dict(case), "capacity": C, "dimp": Dp, "vdimp": Vp}
    # a projection's channels differ in size, a few of them a good deal
    loud = torch.exp(0.5 * normal(D))
    s["q_weight"], s["k_weight"] = 1 + 0.2 * normal(D), (1 + 0.2 * normal(D)) * loud.clamp(max=3)
    s["q_factor"] = torch.full((C,), 1.0 / math.sqrt(D), device="cuda")
    if half:
        angle = torch.arange(C, device="cuda", dtype=torch.float64)[:, None] * torch.pow(10000.0, -torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    s["k_cache"], s["v_cache"] = torch.zeros(G, M, C, Dp, dtype=torch.int8, device="cuda"), torch.zeros(G, C // 32, Vp // 32, 16, 4, 2, 8, dtype=torch.int8, device="cuda")
    s["k_scale"], s["v_scale"] = torch.zeros(G, M, C, device="cuda"), torch.zeros(G, C, device="cuda")
    filled = {"write": 0, "step": first}.get(case["op"], first + n)
    if filled:
        keys = normal(G, M, filled, D) * s["k_weight"]
        numbers, scale = stored(keys)
        s["k_cache"][:, :, :filled, :D], s["k_scale"][:, :, :filled] = numbers.to(torch.int8), scale
        numbers, scale = stored(normal(G, filled, V) * torch.exp(0.3 * normal(G, filled, 1)))
        values = torch.zeros(G, C, Vp, dtype=torch.int8, device="cuda")
        values[:, :filled, :V] = numbers.to(torch.int8)
        s["v_cache"], s["v_scale"][:, :filled] = pack_values(values), scale
    if case["op"] in ("write", "step"):
        t = torch.float32 if case["f32"] or case["op"] == "step" else torch.bfloat16
        parts = [(normal(n, H * M, D) * 1.5, Dp), (normal(n, G * M, D) * loud, Dp), (normal(n, G, V) * torch.exp(0.3 * normal(n, G, 1)), Vp)]
        rows = torch.cat([torch.nn.functional.pad(x, (0, p - x.shape[-1])).reshape(n, -1) for x, p in parts], 1)
        s["rows"] = torch.nn.functional.pad(rows, (0, up_to(rows.shape[1], 64) - rows.shape[1])).to(t).contiguous()
        s["pos"] = torch.tensor([first], dtype=torch.int32, device="cuda")
    if case["op"] == "prompt":
        q = torch.zeros(n, H * M, Dp, device="cuda")
        q[:, :, :D] = normal(n, H * M, D) * s["q_weight"] / math.sqrt(D)
        s["q"] = q.reshape(n, -1).to(torch.bfloat16).contiguous()
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------------
def turned(x, cos, sin):
    """[tokens][heads][columns]: the first pairs of neighbours, by the tables' rows of the tokens"""
    rot = 2 * cos.shape[-1]
    u, v, c, s = x[..., 0:rot:2], x[..., 1:rot:2], cos[:, None], sin[:, None]
    return torch.cat([torch.stack([u * c - v * s, v * c + u * s], -1).flatten(-2), x[..., rot:]], -1)


def projected(s):
    """rows of projections -> queries, keys [tokens][heads][dimp], values [tokens][kv heads][vdimp], in 32 bits"""
    case, Dp, Vp = s["case"], s["dimp"], s["vdimp"]
    H, G, M, D, first, n = (case[k] for k in ("heads", "kv_heads", "maps", "dim", "first", "n"))
    rows = s["rows"].float()
    q, k, v = rows[:, :H * M * Dp].view(n, H * M, Dp), rows[:, H * M * Dp:(H + G) * M * Dp].view(n, G * M, Dp), rows[:, (H + G) * M * Dp:(H + G) * M * Dp + G * Vp].view(n, G, Vp)

    def normed(x, weight):
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS)
        return x * torch.nn.functional.pad(weight, (0, Dp - D))

    q, k = normed(q, s["q_weight"]) * s["q_factor"][first:first + n, None, None], normed(k, s["k_weight"])
    if case["rot"]:
        cos, sin = s["cos"][first:first + n], s["sin"][first:first + n]
        q, k = turned(q, cos, sin), turned(k, cos, sin)
    return q, k, v


def written(s):
    """those keys and values into the cache; the queries, and the values that the cache holds for the tokens: [kv heads][maps][n][dimp], [kv heads][n][vdimp]"""
    case, G, M, first, n = s["case"], s["case"]["kv_heads"], s["case"]["maps"], s["case"]["first"], s["case"]["n"]
    q, k, v = projected(s)
    k, v = k.view(n, G, M, -1).permute(1, 2, 0, 3), v.permute(1, 0, 2)
    kn, ks = stored(k)
    vn, vs = stored(v)
    s["k_cache"][:, :, first:first + n], s["k_scale"][:, :, first:first + n] = kn.to(torch.int8), ks
    p = torch.arange(first, first + n, device="cuda")
    s["v_cache"].permute(0, 1, 4, 6, 2, 5, 3)[:, p // 32, p % 32 // 8, p % 8] = vn.to(torch.int8).view(G, n, -1, 2, 16)
    s["v_scale"][:, first:first + n] = vs
    return q, kn * ks[..., None], vn * vs[..., None]


def held(s, first, n):
    """the cache's values at positions first .. first + n - 1, in 32 bits: keys [kv heads][maps][n][dimp], values [kv heads][n][vdimp]"""
    G, Vp = s["case"]["kv_heads"], s["vdimp"]
    t0, t1 = first // 32, -(-(first + n) // 32)
    values = s["v_cache"][:, t0:t1].permute(0, 1, 4, 6, 2, 5, 3).reshape(G, (t1 - t0) * 32, Vp)[:, first - 32 * t0:first - 32 * t0 + n]
    keys = s["k_cache"][:, :, first:first + n].float() * s["k_scale"][:, :, first:first + n, None]
    return keys, values.float() * s["v_scale"][:, first:first + n, None]


def attended(s, q):
    """q [queries][heads x maps][dimp] of the case's last positions over the cache -> [queries][heads x vdimp]"""
    case = s["case"]
    H, G, M, first, n, V, window = (case[k] for k in ("heads", "kv_heads", "maps", "first", "n", "vdim", "window"))
    begin = max(0, first - window + 1) if window else 0
    keys, values = held(s, begin, first + n - begin)
    q = q.view(n, G, H // G, M, -1).permute(1, 3, 2, 0, 4).reshape(G, M, (H // G) * n, -1)
    scores = torch.matmul(q, keys.transpose(-1, -2).contiguous()).view(G, M, H // G, n, -1)
    p = torch.arange(first, first + n, device="cuda")[:, None]
    j = torch.arange(begin, first + n, device="cuda")[None]
    seen = (j <= p) & (j > p - window) if window else j <= p
    scores = scores.masked_fill(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = weights.sum(-1, keepdim=True)
    a = torch.matmul(weights.view(G, M, (H // G) * n, -1), values[:, None]).view(G, M, H // G, n, -1) / total
    o = a[:, 0]
    if M == 2:
        o = o - LAMBDA * a[:, 1]
        o = o / torch.sqrt(o.square().sum(-1, keepdim=True) / V + EPS) * OUT_SCALE
    return o.permute(2, 0, 1, 3).reshape(n, -1)


def plain(s):
    case = s["case"]
    first, n, op = case["first"], case["n"], case["op"]
    if op == "write":
        q, k, v = written(s)
        return {"q": q.reshape(n, -1).to(s["rows"].dtype), "keys": k.to(torch.bfloat16), "values": v.to(torch.bfloat16)}
    if op == "read":
        t = torch.float32 if case["f32"] else torch.bfloat16
        k, v = held(s, first, n)
        return {"keys": k.to(t), "values": v.to(t)}
    if op == "step":
        q, k, v = written(s)
        return {"out": attended(s, q), "keys": k.to(torch.bfloat16), "values": v.to(torch.bfloat16)}
    return {"out": attended(s, s["q"].float()).to(torch.bfloat16)}


# ---- the framework's calls --------------------------------------------------------------------------------------------
def planned(s):
    """what a program sets up once: the attention's description and the workspaces of its calls"""
    pkg = importlib.import_module("bitnet-rs_amd")
    hip, case = pkg.load(), s["case"]
    hip.init(0)
    H, G, M, D, V, first, n = (case[k] for k in ("heads", "kv_heads", "maps", "dim", "vdim", "first", "n"))
    attn = pkg.Gqa(H, G, M, D, s["dimp"], V, s["vdimp"], s["capacity"], EPS, LAMBDA, OUT_SCALE, s["q_weight"].data_ptr(), s["k_weight"].data_ptr(), s["q_factor"].data_ptr(),
                   s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), rot_dims=case["rot"], window=case["window"])
    if case["rot"]:
        attn.rope_cos, attn.rope_sin = s["cos"].data_ptr(), s["sin"].data_ptr()
    scratch = 0
    if case["op"] == "step":
        scratch = hip.gqa_scratch_bytes(H, M, s["vdimp"], 1)
    elif case["op"] == "prompt":
        scratch = hip.kv8_prefill_scratch_bytes(attn, first + n, n)
    return hip, attn, torch.empty(scratch, dtype=torch.uint8, device="cuda") if scratch else None


def called(s):
    if "plan" not in s:
        s["plan"] = planned(s)
    hip, attn, scratch = s["plan"]
    case, ks, vs = s["case"], s["k_scale"], s["v_scale"]
    H, G, M, first, n, op = (case[k] for k in ("heads", "kv_heads", "maps", "first", "n", "op"))

    def new(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    out = {}
    if op == "write":
        out["q"] = new(n, H * M * s["dimp"], dtype=s["rows"].dtype)
        hip.kv8_rows_dev(attn, ks, vs, s["rows"], s["rows"].shape[1], case["f32"], s["pos"], n, out["q"], H * M * s["dimp"])
    elif op == "step":
        out["out"] = new(1, H * s["vdimp"], dtype=torch.float32)
        hip.kv8_step_dev(attn, ks, vs, s["rows"], s["pos"], scratch)
        hip.gqa_merge_dev(attn, s["pos"], 0, 1, scratch, out["out"], H * s["vdimp"], False)
    elif op == "prompt":
        out["out"] = new(n, H * s["vdimp"])
        hip.kv8_prefill_dev(attn, ks, vs, s["q"], s["q"].shape[1], first + n, n, out["out"], H * s["vdimp"], scratch, scratch.numel() if scratch is not None else 0)
        return out
    f32 = op == "read" and case["f32"]
    out["keys"], out["values"] = (new(*shape, dtype=torch.float32 if f32 else torch.bfloat16) for shape in ((G, M, n, s["dimp"]), (G, n, s["vdimp"])))
    hip.kv8_read_dev(attn, ks, vs, first, n, out["keys"], out["values"], f32)
    return out


def run(state):
    return called(state) if own else plain(state)


# ---- by definition, in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    H, G, M, D, V, first, n = (case[k] for k in ("heads", "kv_heads", "maps", "dim", "vdim", "first", "n"))
    Dp, Vp, group = s["dimp"], s["vdimp"], H // G

    def quantised(x):
        a = x.abs().max(-1, keepdim=True).values
        return torch.where(a > 0, torch.round(x * 127 / a) * (a / 127), torch.zeros_like(x))

    def cached(kv):
        """keys [maps][capacity][dimp] and values [capacity][vdimp] of a kv head"""
        c, p = torch.arange(Vp, device="cuda"), torch.arange(s["capacity"], device="cuda")[:, None]
        at = ((p // 32 * (Vp // 32) + c // 32) * 16 + c % 16) * 64 + p % 32 // 8 * 16 + c % 32 // 16 * 8 + p % 8
        return s["k_cache"][kv].to(f64) * s["k_scale"][kv, :, :, None].to(f64), s["v_cache"][kv].reshape(-1)[at].to(f64) * s["v_scale"][kv, :, None].to(f64)

    def finished(x, weight, factor=None):
        """[n][heads][dimp]: norm, weight, factor, rotation"""
        x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt()
        x[..., :D] *= weight.to(f64)
        if factor is not None:
            x = x * factor.to(f64)[:, None, None]
        half = case["rot"] // 2
        if half:
            z = torch.view_as_complex(x[..., :2 * half].reshape(n, -1, half, 2).contiguous())
            z = z * torch.complex(s["cos"][first:first + n].to(f64), s["sin"][first:first + n].to(f64))[:, None]
            x = torch.cat([torch.view_as_real(z).reshape(n, -1, 2 * half), x[..., 2 * half:]], -1)
        return x

    out = {}
    if case["op"] in ("write", "step"):
        rows = s["rows"].to(f64)
        q = finished(rows[:, :H * M * Dp].reshape(n, H * M, Dp), s["q_weight"], s["q_factor"][first:first + n])
        keys = quantised(finished(rows[:, H * M * Dp:(H + G) * M * Dp].reshape(n, G * M, Dp), s["k_weight"])).reshape(n, G, M, Dp)
        values = quantised(rows[:, (H + G) * M * Dp:(H + G) * M * Dp + G * Vp].reshape(n, G, Vp))
        out["keys"], out["values"] = keys.permute(1, 2, 0, 3).contiguous(), values.permute(1, 0, 2).contiguous()
        if case["op"] == "write":
            out["q"] = q.reshape(n, -1)
            return out
    if case["op"] == "read":
        both = [cached(kv) for kv in range(G)]
        return {"keys": torch.stack([k[:, first:first + n] for k, _ in both]), "values": torch.stack([v[first:first + n] for _, v in both])}
    if case["op"] == "prompt":
        q = s["q"].to(f64).reshape(n, H * M, Dp)
    result = torch.zeros(n, H, Vp, dtype=f64, device="cuda")
    here = torch.arange(first, first + n, device="cuda")[:, None]
    there = torch.arange(first + n, device="cuda")[None]
    hidden = there > here
    if case["window"]:
        hidden |= there <= here - case["window"]
    for kv in range(G):
        k, v = cached(kv)
        if case["op"] == "step":
            k[:, first], v[first] = out["keys"][kv, :, 0], out["values"][kv, 0]
        for h in range(kv * group, (kv + 1) * group):
            each = []
            for m in range(M):
                z = q[:, h * M + m] @ k[m, :first + n].T
                z.masked_fill_(hidden, -math.inf)
                each.append(torch.softmax(z, -1) @ v[:first + n])
            o = each[0]
            if M == 2:
                o = each[0] - LAMBDA * each[1]
                o = OUT_SCALE * o / (o.square().sum(-1, keepdim=True) / V + EPS).sqrt()
            result[:, h] = o
    out["out"] = result.reshape(n, -1)
    return out
