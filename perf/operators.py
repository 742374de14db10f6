"""Cases of the 8-bit key/value cache and of the rotary forms: what is computed, on which inputs, in a plain form.

Four operators of one decoder layer over a paged cache (blocks of `bs` slots, a block table a row):

  write  rotate q and k of a fused q/k/v projection and store k and v in the cache, in the inputs' type
  store  the same with a cache of e4m3 codes and one fp32 scale for each (slot, KV head)
  read   the keys and values of a quantised cache as dense bf16 or fp32 tensors, as attention of many queries reads them
  attend one query a row against a quantised cache (grouped heads, slots up to the row's position)

Rotation of a pair (a, b) by its position's (c, s): (a c - b s, b c + a s). The pairs are (x[i], x[i + r/2]) in the
"half" layout and (x[2i], x[2i+1]) in the "interleaved" one, i < r/2; values from r on are copied. A row (slot, head) of
the quantised cache has scale = max(largest |x| / 448, 2^-126) and codes e4m3(x / scale). A negative position marks
padding: a token that writes nothing, a query whose output is zero.
"""

import math

import torch

own = False

F8 = torch.float8_e4m3fn
TINY = 2.0 ** -126
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------- cases

def _write(name, op, B, T, nh, nkv, hd, rd, layout, scaling, start, bs, dtype, ragged):
    return {"name": name, "op": op, "B": B, "T": T, "nh": nh, "nkv": nkv, "hd": hd, "rd": rd, "layout": layout,
            "scaling": scaling, "start": start, "bs": bs, "dtype": dtype, "ragged": ragged}


def _read(name, B, slots, nkv, hd, bs, dtype):
    return {"name": name, "op": "read", "B": B, "slots": slots, "nkv": nkv, "hd": hd, "bs": bs, "dtype": dtype}


def _attend(name, B, ctx, nh, nkv, hd, bs, dtype, padded):
    return {"name": name, "op": "attend", "B": B, "ctx": ctx, "nh": nh, "nkv": nkv, "hd": hd, "bs": bs, "dtype": dtype,
            "padded": padded}


def listed():
    return [
        # one sequence's next token at a far position, half of each head rotated by neighbouring pairs: latency counts
        _write("write-token", "write", 1, 1, 32, 8, 128, 64, "interleaved", "by_parts", 9001, 16, "bf16", False),
        # four prompts of one micro-batch, the 8B shape, whole heads, angles stretched for a long context
        _write("write-prompts", "write", 4, 2048, 32, 8, 128, 128, "half", "ntk", 0, 16, "bf16", False),
        # fp32 parity runs: an odd batch continued in the middle of a block, head size off the vector widths, padded rows
        _write("write-odd-fp32", "write", 3, 257, 9, 3, 80, 20, "interleaved", "linear", 77, 16, "fp32", True),
        # a decode step of a full batch into the 8-bit cache
        _write("store-batch", "store", 64, 1, 32, 8, 128, 128, "half", "none", 4095, 16, "bf16", True),
        # prompts of the 70B shape into the 8-bit cache: the largest write
        _write("store-prompts", "store", 8, 2048, 64, 8, 128, 128, "half", "by_parts", 0, 16, "bf16", True),
        # an fp32 chunk of a prompt, partial rotation, odd lengths and blocks
        _write("store-odd-fp32", "store", 5, 131, 10, 5, 96, 48, "half", "ntk", 1000, 24, "fp32", True),
        # a short prompt's cache read back for its attention
        _read("read-short", 1, 300, 8, 128, 16, "bf16"),
        # long prompts read back for the attention of their next chunk: the largest read
        _read("read-long", 8, 16384, 8, 128, 16, "bf16"),
        # one short conversation's next token: latency counts
        _attend("attend-short", 1, 48, 32, 8, 128, 16, "bf16", False),
        # a decode step of 64 running requests of mixed lengths
        _attend("attend-batch", 64, 4352, 32, 8, 128, 16, "bf16", True),
        # two long documents, 64 query heads
        _attend("attend-long", 2, 131072, 64, 8, 128, 64, "bf16", False),
        # fp32 parity runs: every head its own keys, blocks that end inside any tile
        _attend("attend-odd-fp32", 7, 1500, 12, 12, 64, 20, "fp32", True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    op = rng.choice(("write", "store", "read", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    hd = rng.choice((128, 128, 64, 64, 256, 32, 80, 96, 112))
    nkv = _log(rng, 1, 12)
    bs = rng.choice((16, 16, 32, 64, 8, 20, 1, 48, 256))
    if op in ("write", "store"):
        T = _log(rng, 1, 3000)
        B = _log(rng, 1, max(1, min(96, 16000 // T)))
        rd = rng.choice((hd, hd, hd // 2, hd // 4 * 2, 16, hd - 2))
        layout, scaling = rng.choice(("half", "interleaved")), rng.choice(("none", "linear", "ntk", "by_parts"))
        rep = rng.choice((1, 2, 4, 8, 5))
        while B * T * nkv * (rep + 2) * hd > 8192 * 80 * 128:
            B, T = max(1, B // 2), max(1, T * 3 // 4)
        c = _write("", op, B, T, nkv * rep, nkv, hd, rd, layout, scaling, rng.choice((0, _log(rng, 1, 30000))), bs, dtype,
                   rng.random() < 0.5)
    elif op == "read":
        slots = _log(rng, 1, 40000)
        B = _log(rng, 1, 64)
        while B * slots * nkv * hd > 70000000:
            B, slots = max(1, B // 2), max(1, slots * 3 // 4)
        c = _read("", B, slots, nkv, hd, bs, dtype)
    else:
        ctx = _log(rng, 1, 100000)
        B = _log(rng, 1, 96)
        while B * ctx * nkv * hd > 270000000:
            B, ctx = max(1, B // 2), max(1, ctx * 3 // 4)
        c = _attend("", B, ctx, nkv * rng.choice((1, 2, 4, 4, 7, 8, 16)), nkv, hd, bs, dtype, rng.random() < 0.5)
    c.pop("name")
    return c


def _tokens(case):
    """Real tokens of each row: the rows of a ragged batch hold different numbers, its last one half (none of one)."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    return [T - (i * 37) % (T // 2 + 1) if i < B - 1 or B < 3 else T // 2 for i in range(B)]


def _starts(case):
    """Each row's first position: rows of a batch stand at different places, the first one furthest."""
    return [max(0, case["start"] - 13 * (i % 8)) for i in range(case["B"])]


def _visible(case):
    """Visible slots of each row; a padded batch ends in a row that sees none."""
    B, ctx = case["B"], case["ctx"]
    n = [ctx - (i * 977) % (ctx // 2 + 1) for i in range(B)]
    if case["padded"] and B > 1:
        n[-1] = 0
    return n


def work(case):
    el = 2 if case.get("dtype") == "bf16" else 4
    nkv, hd = case["nkv"], case["hd"]
    if case["op"] in ("write", "store"):
        n = _tokens(case)
        starts = _starts(case)
        tokens, nh, rd = sum(n), case["nh"], case["rd"]
        rows = len(set().union(*(range(s, s + t) for s, t in zip(starts, n))))
        blocks = sum(-(-(s % case["bs"] + t) // case["bs"]) for s, t in zip(starts, n) if t)
        kv = 2 * nkv * hd * el if case["op"] == "write" else 2 * nkv * (hd + 4)
        return {"bytes": tokens * ((2 * nh + 2 * nkv) * hd * el + kv) + case["B"] * case["T"] * 8 + rows * rd * 4 + blocks * 8,
                "flops": tokens * ((nh + nkv) * rd * 3 + (4 * nkv * hd if case["op"] == "store" else 0))}
    if case["op"] == "read":
        n = case["B"] * case["slots"] * nkv
        return {"bytes": 2 * n * (hd + 4 + hd * el) + case["B"] * -(-case["slots"] // case["bs"]) * 8, "flops": 2 * n * hd}
    vis, nh = _visible(case), case["nh"]
    return {"bytes": sum(vis) * nkv * 2 * (hd + 4) + 2 * case["B"] * nh * hd * el
            + sum(-(-v // case["bs"]) for v in vis) * 8 + case["B"] * 8,
            "flops": 4 * sum(vis) * nh * hd}


# ------------------------------------------------------------------------------------------------ inputs

def _frequencies(rd, scaling, device):
    """Angle a position of each pair, in 64 bits, and the factor on cos and sin."""
    i = torch.arange(0, rd, 2, dtype=torch.float64, device=device)
    theta, factor, original = 500000.0, 8.0, 8192.0
    if scaling == "ntk" and rd > 2:      # a larger base: the fastest pair keeps its angle, the slowest is stretched
        theta = theta * factor ** (rd / (rd - 2))
    f = theta ** (-i / rd)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "by_parts":            # pairs that turn often within the original length keep their angle
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1
    return f, 1.0


def _table(B, cols, spare, g, device):
    """Each row's blocks, in no order, none used twice, and how many blocks the pool has."""
    n = B * cols + spare
    return torch.randperm(n, generator=g, device=device)[:B * cols].view(B, cols), n


def _codes(shape, g, device):
    """Codes as a store leaves them: most of the range used, a few at its ends."""
    x = torch.empty(shape, dtype=torch.bfloat16, device=device).normal_(0, 130, generator=g)
    return x.clamp_(-448, 448).to(F8)


def _scales(shape, g, device):
    """Scales of rows whose values are near 1, some rows several times larger than others."""
    return torch.empty(shape, device=device).normal_(0, 0.4, generator=g).exp_().mul_(0.0075)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    B, nkv, hd, bs = case["B"], case["nkv"], case["hd"], case["bs"]
    s = {"case": case}
    if case["op"] in ("write", "store"):
        T, nh, rd = case["T"], case["nh"], case["rd"]
        n, starts = _tokens(case), _starts(case)
        cols = -(-(max(starts) + T) // bs)
        # only the blocks that the tokens fall into are the row's own; earlier columns repeat its first one of these
        lo = min(starts) // bs
        own_blocks, total = _table(B, cols - lo, 3, g, dev)
        s["table"] = torch.cat([own_blocks[:, :1].expand(B, lo), own_blocks], 1).contiguous()
        j = torch.arange(T, device=dev)
        pos = torch.tensor(starts, device=dev)[:, None] + j
        real = j < torch.tensor(n, device=dev)[:, None]
        s["positions"] = torch.where(real, pos, -1).contiguous()
        s["row"], s["col"] = torch.nonzero(real, as_tuple=True)      # a program that made the batch has them at hand
        f, m = _frequencies(rd, case["scaling"], dev)
        a = torch.arange(max(starts) + T, dtype=torch.float64, device=dev)[:, None] * f
        s["cos"], s["sin"] = (a.cos() * m).float(), (a.sin() * m).float()
        x = torch.empty(B * T, (nh + 2 * nkv) * hd, device=dev).normal_(generator=g)
        x *= torch.empty(x.shape[1], device=dev).normal_(0, 0.5, generator=g).exp_()     # some channels are larger
        s["qkv"] = x.to(dt)
        s["q"] = torch.zeros(B * T, nh * hd, dtype=dt, device=dev)
        shape = (total, nkv, bs, hd)
        if case["op"] == "write":
            s["k"] = torch.empty(shape, dtype=dt, device=dev).normal_(generator=g)
            s["v"] = torch.empty(shape, dtype=dt, device=dev).normal_(generator=g)
            return s
    elif case["op"] == "read":
        s["table"], total = _table(B, -(-case["slots"] // bs), 3, g, dev)
        shape = (total, nkv, bs, hd)
    else:
        nh, vis = case["nh"], _visible(case)
        s["table"], total = _table(B, -(-case["ctx"] // bs), 3, g, dev)
        shape = (total, nkv, bs, hd)
        s["positions"] = torch.tensor(vis, device=dev) - 1
        s["q"] = (torch.empty(B, nh * hd, device=dev).normal_(generator=g) * 1.5).to(dt)
        s["out"] = torch.empty(B, nh * hd, dtype=dt, device=dev)
    s["k"], s["v"] = _codes(shape, g, dev), _codes(shape, g, dev)
    s["k_scale"], s["v_scale"] = _scales(shape[:3], g, dev), _scales(shape[:3], g, dev)
    return s


# -------------------------------------------------------------------------------------------- plain form

def _rotate(x, cos, sin, layout):
    """x (n, heads, hd) fp32, cos and sin (n, r/2)."""
    r, c, s = 2 * cos.shape[1], cos[:, None], sin[:, None]
    if layout == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_write(s):
    c = s["case"]
    nh, nkv, hd, bs, dt = c["nh"], c["nkv"], c["hd"], c["bs"], TYPES[c["dtype"]]
    row, col = s["row"], s["col"]
    p, tok = s["positions"][row, col], row * c["T"] + col
    x = s["qkv"][tok].float().view(-1, nh + 2 * nkv, hd)
    qk = _rotate(x[:, :nh + nkv], s["cos"][p], s["sin"][p], c["layout"])
    s["q"][tok] = qk[:, :nh].flatten(1).to(dt)
    block, slot = s["table"][row, p // bs], p % bs
    k, v = qk[:, nh:], x[:, nh + nkv:]
    if c["op"] == "write":
        s["k"][block, :, slot] = k.to(dt)
        s["v"][block, :, slot] = v.to(dt)
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    ks, vs = ((y.abs().amax(-1) / 448).clamp_min(TINY) for y in (k, v))
    s["k"].view(torch.uint8)[block, :, slot] = (k / ks[..., None]).to(F8).view(torch.uint8)
    s["v"].view(torch.uint8)[block, :, slot] = (v / vs[..., None]).to(F8).view(torch.uint8)
    s["k_scale"][block, :, slot] = ks
    s["v_scale"][block, :, slot] = vs
    return {"q": s["q"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _dense(codes, scale, table, slots):
    """(B, nkv, slots, hd) fp32 of a quantised pool."""
    B, nkv, hd = table.shape[0], codes.shape[1], codes.shape[3]
    x = codes.view(torch.uint8)[table].view(F8).float() * scale[table][..., None]
    return x.transpose(1, 2).reshape(B, nkv, -1, hd)[:, :, :slots]


def _plain_read(s):
    c = s["case"]
    dt = TYPES[c["dtype"]]
    return {"k": _dense(s["k"], s["k_scale"], s["table"], c["slots"]).to(dt).contiguous(),
            "v": _dense(s["v"], s["v_scale"], s["table"], c["slots"]).to(dt).contiguous()}


def _plain_attend(s):
    c = s["case"]
    B, nh, nkv, hd, ctx = c["B"], c["nh"], c["nkv"], c["hd"], c["ctx"]
    q = s["q"].float().view(B, nkv, nh // nkv, hd) / math.sqrt(hd)
    score = q @ _dense(s["k"], s["k_scale"], s["table"], ctx).transpose(2, 3)
    seen = (torch.arange(ctx, device=q.device) <= s["positions"][:, None])[:, None, None]
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.where(seen, (score - top).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    o = e @ _dense(s["v"], s["v_scale"], s["table"], ctx) / torch.where(seen.any(-1, keepdim=True), total, 1.0)
    return {"out": o.view(B, nh * hd).to(TYPES[c["dtype"]])}


# ------------------------------------------------------------------------------------ the framework's calls

def _own(s):
    from forgeserve_b200 import ops

    c = s["case"]
    if c["op"] == "write":
        ops.rotary_kv_write(s["qkv"], s["cos"], s["sin"], s["positions"], ops.paged_desc(s["k"], s["v"], s["table"]),
                            c["B"], c["T"], c["nh"], c["nkv"], c["hd"], layout=c["layout"], q_out=s["q"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    kv = ops.quant_paged_desc(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"])
    if c["op"] == "store":
        ops.rotary_kv_write(s["qkv"], s["cos"], s["sin"], s["positions"], kv, c["B"], c["T"], c["nh"], c["nkv"], c["hd"],
                            layout=c["layout"], q_out=s["q"])
        return {"q": s["q"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["op"] == "read":
        k, v = ops.kv_dequant(kv, c["B"], c["slots"], c["nkv"], c["hd"], TYPES[c["dtype"]])
        return {"k": k, "v": v}
    return {"out": ops.attention_decode_quant(s["q"], kv, c["ctx"], s["positions"], s["out"], c["B"], c["nh"], c["nkv"],
                                              c["hd"])}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_read(state) if op == "read" else _plain_attend(state) if op == "attend" else _plain_write(state)


# ------------------------------------------------------------------------------------- 64 bits, row by row

def _exact_write(s):
    c = s["case"]
    T, nh, nkv, hd, bs = c["T"], c["nh"], c["nkv"], c["hd"], c["bs"]
    r = 2 * s["cos"].shape[1]
    first = torch.arange(r // 2, device="cuda") * (2 if c["layout"] == "interleaved" else 1)
    second = first + (1 if c["layout"] == "interleaved" else r // 2)
    out = {n: s[n].double() for n in ("q", "k", "v", "k_scale", "v_scale") if n in s}
    for row in range(c["B"]):
        p = s["positions"][row]
        p = p[p >= 0]
        if not p.numel():
            continue
        z = s["qkv"][row * T:row * T + p.numel()].double().view(-1, nh + 2 * nkv, hd)
        co, si = s["cos"].double()[p][:, None, :], s["sin"].double()[p][:, None, :]
        y = z.clone()
        y[:, :nh + nkv, first] = z[:, :nh + nkv, first] * co - z[:, :nh + nkv, second] * si
        y[:, :nh + nkv, second] = z[:, :nh + nkv, second] * co + z[:, :nh + nkv, first] * si
        out["q"][row * T:row * T + p.numel()] = y[:, :nh].reshape(p.numel(), -1)
        block, slot = s["table"][row][torch.div(p, bs, rounding_mode="floor")], p.remainder(bs)
        for n, part in (("k", y[:, nh:nh + nkv]), ("v", y[:, nh + nkv:])):
            if c["op"] == "store":
                scale = torch.maximum(part.abs().max(-1).values / 448.0, torch.tensor(TINY, dtype=torch.float64, device="cuda"))
                out[n + "_scale"][block, :, slot] = scale
                part = part / scale[..., None]      # the value that the code is rounded from
            out[n][block, :, slot] = part
    return out


def _exact_row(s, name, row, slots):
    """One row's keys or values, (nkv, slots, hd) in 64 bits."""
    t = torch.arange(slots, device="cuda")
    block, slot = s["table"][row][t // s["case"]["bs"]], t % s["case"]["bs"]
    code = s[name].view(torch.uint8)[block, :, slot].view(F8).double()
    return (code * s[name + "_scale"][block, :, slot].double()[..., None]).permute(1, 0, 2)


def _exact_read(s):
    c = s["case"]
    return {n: torch.stack([_exact_row(s, n, row, c["slots"]) for row in range(c["B"])]) for n in ("k", "v")}


def _exact_attend(s):
    c = s["case"]
    rep, hd = c["nh"] // c["nkv"], c["hd"]
    out = torch.zeros(c["B"], c["nh"] * hd, dtype=torch.float64, device="cuda")
    for row, n in enumerate(_visible(c)):
        if n:
            k, v = _exact_row(s, "k", row, n), _exact_row(s, "v", row, n)
            q = s["q"][row].double().view(c["nkv"], rep, hd)
            p = torch.softmax(torch.einsum("grd,gsd->grs", q, k) / hd ** 0.5, -1)
            out[row] = torch.einsum("grs,gsd->grd", p, v).reshape(-1)
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_read(s) if case["op"] == "read" else _exact_attend(s) if case["op"] == "attend" else _exact_write(s)
