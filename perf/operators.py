"""Products of many rows with packed organs, as timed cases.

Rows of a batch (tokens, requests) are grouped by an id, an expert or an
adapter, and multiplied with the packed matrix of their group:

  * group    ids -> each group's range, the stable order of the rows and its inverse
  * product  y_i = W_g x_i for the rows i of every group g (a routed down projection)
  * swiglu   y_i = silu(G_g x_i) * (U_g x_i) (the routed gate and up projections)
  * combine  y_t = base_t + sum_r w_tr x[pos_tr] (the routed outputs of a token, weighted)
  * lora     y_t = W x_t + s_a B_a (A_a x_t) with the adapter a of each row

`own` selects the framework's kernels; without it every operator is computed
in its plain form: weights decoded to f32, f32 products, one rounding.
Weights are N(0, 0.02) draws quantized to the organ's format, x is N(0, 1).
"""
from __future__ import annotations

import ctypes as C
import math
from types import SimpleNamespace

import torch

own = False

SIGMA = 0.02
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a decode step of 64 requests: eight experts each, of 256
        dict(name="group_64x8_of_256", op="group", tokens=64, per_row=8, groups=256, absent=0.0),
        # a long prefill's routes: ten of 512 experts for 32768 tokens, some of them padding
        dict(name="group_32768x10_of_512", op="group", tokens=32768, per_row=10, groups=512, absent=0.02),
        # decode of 16 requests: nearly every routed row has an expert of its own, weights bound it
        dict(name="swiglu_q4_16x10_of_512", op="swiglu", kind="q4", group=32, rows=512, cols=2048, groups=512,
             tokens=16, per_row=10, x="f32", y="f32", absent=0.0),
        # prefill of 4096 tokens through 512 small experts: about 80 rows each
        dict(name="swiglu_q4_4096x10_of_512", op="swiglu", kind="q4", group=32, rows=512, cols=2048, groups=512,
             tokens=4096, per_row=10, x="bf16", y="bf16", absent=0.0),
        # one rank's 32 of a wide model's 256 experts, the rows that a large prefill sends it
        dict(name="swiglu_q4_8192_of_32_wide", op="swiglu", kind="q4", group=32, rows=2048, cols=7168, groups=32,
             tokens=8192, per_row=1, x="bf16", y="bf16", absent=0.0),
        # the down projection of a decode step of 64 requests in the mixed format
        dict(name="product_mixed_64x10_of_512", op="product", kind="mixed", group=128, rows=2048, cols=512, groups=512,
             tokens=64, per_row=10, x="bf16", y="f32", absent=0.0),
        # the down projection of the 4096-token prefill
        dict(name="product_q4_4096x10_of_512", op="product", kind="q4", group=32, rows=2048, cols=512, groups=512,
             tokens=4096, per_row=10, x="bf16", y="bf16", absent=0.0),
        # the weighted sum at the end of a routed block: 32 requests of a wide model ...
        dict(name="combine_32x8x7168", op="combine", cols=7168, tokens=32, per_row=8, x="f32", y="f32", absent=0.0),
        # ... and a prefill, padding among the tokens
        dict(name="combine_8192x10x2048", op="combine", cols=2048, tokens=8192, per_row=10, x="bf16", y="bf16",
             absent=0.02),
        # one token of one request with an adapter: latency
        dict(name="lora_q8_1x2048x2048_r16", op="lora", kind="q8", group=64, rows=2048, cols=2048, tokens=1, slots=4,
             rank=16, requests=1, x="f32", y="f32", absent=0.0),
        # a decode step of 64 requests over 32 adapters, some requests without one
        dict(name="lora_q4_64x4096x2048_r32", op="lora", kind="q4", group=32, rows=4096, cols=2048, tokens=64,
             slots=32, rank=32, requests=64, x="bf16", y="bf16", absent=0.1),
        # prefill of eight requests with an adapter each through a wide projection
        dict(name="lora_q4_4096x2048x7168_r64", op="lora", kind="q4", group=32, rows=2048, cols=7168, tokens=4096,
             slots=8, rank=64, requests=8, x="bf16", y="bf16", absent=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case over the ranges the listed ones stand for."""
    op = rng.choice(("group", "swiglu", "swiglu", "product", "product", "combine", "lora", "lora"))
    absent = rng.choice((0.0, 0.0, 0.05))
    if op == "group":
        per_row = rng.randint(1, 10)
        return dict(op=op, tokens=max(1, _log(rng, 8, 327680) // per_row), per_row=per_row,
                    groups=_log(rng, 2, 1024), absent=absent)
    types = rng.choice((("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("f16", "f16"), ("f32", "bf16")))
    if op == "combine":
        return dict(op=op, cols=_log(rng, 100, 8192), tokens=_log(rng, 1, 8192), per_row=rng.randint(1, 10),
                    x=types[0], y=types[1], absent=absent)
    kind = rng.choice(("q4", "q4", "q4", "q8", "bin", "mixed", "u3"))
    group = {"q4": rng.choice((32, 64, 128)), "q8": 64, "u3": 64}.get(kind, 128)
    unit = 32 if kind == "u3" else group
    rows, cols = _log(rng, 60, 4096), unit * max(1, _log(rng, 256, 7168) // unit)
    if op == "lora":
        tokens, slots = _log(rng, 1, 4096), rng.randint(1, 32)
        return dict(op=op, kind=kind, group=group, rows=rows, cols=cols, tokens=tokens, slots=slots,
                    rank=rng.choice((4, 8, 16, 24, 32, 64)), requests=min(tokens, rng.choice((1, 4, 16, 64))),
                    x=types[0], y=types[1], absent=absent)
    groups = max(2, min(_log(rng, 4, 512), (1 << 30) // (rows * cols)))
    per_row = rng.randint(1, min(10, groups)) if op == "swiglu" else 1
    most = max(64, (1 << 36) // (rows * cols))
    tokens = max(1, _log(rng, 1, min(32768, most)) // per_row)
    return dict(op=op, kind=kind, group=group, rows=rows, cols=cols, groups=groups, tokens=tokens, per_row=per_row,
                x=types[0], y=types[1], absent=absent)


# ---------------------------------------------------------------- inputs

def _gen(seed, tag):
    return torch.Generator("cuda").manual_seed((seed * 1000003 + tag) & 0x7FFFFFFFFFFF)


def _randn(seed, tag, *shape):
    return torch.randn(*shape, generator=_gen(seed, tag), device="cuda", dtype=torch.float32)


def _rand(seed, tag, *shape):
    return torch.rand(*shape, generator=_gen(seed, tag), device="cuda", dtype=torch.float32)


def _codes(kind, group, seed, tag, n, rows, cols):
    """n matrices of N(0, 0.02) weights quantized: integer codes [n, rows, cols] (uint8), f16 scales, and for the
    mixed kind which groups of 128 are binary.  The scale of an element is scales[matrix, flat index // unit]."""
    w = _randn(seed, tag, n, rows * cols) * SIGMA
    if kind == "u3" and (rows * cols) % 64:
        w = torch.nn.functional.pad(w, (0, 64 - (rows * cols) % 64))
    if kind in ("q4", "q8", "u3"):
        top = {"q4": 7, "q8": 127, "u3": 3}[kind]
        low = {"q4": -8, "q8": -127, "u3": -3}[kind]
        g = w.view(n, -1, group)
        s = (g.abs().amax(-1) / top).to(torch.float16)
        q = (g / s.float().unsqueeze(-1)).round_().clamp_(low, top).sub_(low).to(torch.uint8)
        return q.view(n, -1), s, None
    g = w.view(n, -1, 128)
    sb = g.abs().mean(-1).to(torch.float16)
    b = (g > 0).to(torch.uint8)
    if kind == "bin":
        return b.view(n, -1), sb, None
    coin = _rand(seed, tag + 1, n, g.shape[1]) < 0.7
    h = w.view(n, -1, 64)
    s2 = (h.abs().mean(-1) * 1.25).to(torch.float16).view(n, -1, 2)
    c = (h / s2.view(n, -1).float().unsqueeze(-1) + 1.5).round_().clamp_(0, 3).to(torch.uint8).view(n, -1, 128)
    code = torch.where(coin.unsqueeze(-1), b, c).view(n, -1)
    scale = torch.where(coin.unsqueeze(-1), sb.unsqueeze(-1).expand(-1, -1, 2), s2).reshape(n, -1).contiguous()
    return code, scale, coin


def _bits(v, width):
    """The low `width` bits of every value of v [n, m], LSB first, in bytes (m * width a multiple of 8)."""
    shifts = torch.arange(width, device=v.device, dtype=torch.uint8)
    b = ((v.unsqueeze(-1) >> shifts) & 1).view(v.shape[0], -1, 8)
    return (b << torch.arange(8, device=v.device, dtype=torch.uint8)).sum(-1, dtype=torch.uint8)


def _pack(kind, code, scale, coin):
    """The organ's bytes: what a file of it holds, for n matrices at once."""
    n = code.shape[0]
    p = SimpleNamespace(kind=kind)
    if kind == "mixed":
        c = code.view(n, -1, 128)
        s = scale.view(n, -1, 2)
        p.tags = [_bits(torch.nn.functional.pad(t.to(torch.uint8).unsqueeze(0), (0, -t.numel() % 8)), 1)[0] for t in coin]
        p.bin_scales = [s[i, coin[i], 0].contiguous() for i in range(n)]
        p.bin_signs = [_bits(c[i, coin[i]].reshape(1, -1), 1)[0] for i in range(n)]
        p.q2_scales = [s[i, ~coin[i]].reshape(-1).contiguous() for i in range(n)]
        p.q2_codes = [_bits(c[i, ~coin[i]].reshape(1, -1), 2)[0] for i in range(n)]
        return p
    p.scales = scale
    p.codes = (code[:, 0::2] | (code[:, 1::2] << 4)) if kind == "q4" else code.clone() if kind == "q8" else \
        _bits(code, 1 if kind == "bin" else 3)
    return p


def _ids(c, seed):
    """Routes of a batch: a router's choices, some groups much busier than others, the ids of one token distinct;
    `absent` is the share of tokens that are padding (id -1)."""
    t, k, g = c["tokens"], c["per_row"], c["groups"]
    bias = _randn(seed, 1, g) * 0.5
    gumbel = -torch.log(-torch.log(_rand(seed, 2, t, g).clamp_(1e-20, 1 - 1e-7)))
    ids = (gumbel + bias).topk(min(k, g), dim=1).indices.to(torch.int32)
    if k > g:
        ids = ids.repeat(1, -(-k // g))[:, :k].contiguous()
    ids[_rand(seed, 3, t) < c["absent"]] = -1
    return ids.reshape(-1)


def _grouping(ids, groups):
    key = torch.where((ids >= 0) & (ids < groups), ids, groups).long()
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(groups + 1, device=ids.device))  # keys below each group
    return offsets.to(torch.int32), order.to(torch.int32)


def _adapter_ids(c, seed):
    """Rows of `requests` requests, one after the other, each with its adapter (or none)."""
    t, r = c["tokens"], c["requests"]
    adapter = (_rand(seed, 4, r) * c["slots"]).to(torch.int32)
    adapter[_rand(seed, 5, r) < c["absent"]] = -1
    edge = torch.cat([torch.zeros(1, device="cuda"), _rand(seed, 6, r - 1).sort().values]) * t if t > r else \
        torch.arange(r, device="cuda")
    row = torch.arange(t, device="cuda")
    request = (torch.searchsorted(edge.contiguous(), row.to(edge.dtype), right=True) - 1).clamp_(0, r - 1)
    return adapter[request].contiguous()


def _inputs(c, seed):
    """Everything of a case but the framework's handles, on the GPU."""
    s = SimpleNamespace(c=c)
    op = c["op"]
    if op == "group":
        s.ids = _ids(c, seed)
        return s
    if op == "combine":
        n = c["tokens"] * c["per_row"]
        s.x = _randn(seed, 10, n, c["cols"]).to(DTYPES[c["x"]])
        s.base = _randn(seed, 11, c["tokens"], c["cols"]).to(DTYPES[c["y"]])  # the residual that the sum is added to
        s.y = torch.zeros_like(s.base)
        w = _rand(seed, 12, c["tokens"], c["per_row"]) + 0.05
        s.w = w / w.sum(1, keepdim=True)
        pos = torch.randperm(n, generator=_gen(seed, 13), device="cuda").to(torch.int32).view(c["tokens"], -1)
        pos[_rand(seed, 14, c["tokens"]) < c["absent"]] = -1
        s.pos = pos.contiguous()
        return s
    n_rows = c["tokens"]
    if op == "lora":
        s.ids = _adapter_ids(c, seed)
        s.offsets, s.order = _grouping(s.ids, c["slots"])
        s.codes = _codes(c["kind"], c["group"], seed, 20, 1, c["rows"], c["cols"])
        s.a = (_randn(seed, 30, c["slots"], c["rank"], c["cols"]) / math.sqrt(c["cols"])).to(torch.bfloat16)
        s.b = (_randn(seed, 31, c["slots"], c["rows"], c["rank"]) * SIGMA).to(torch.bfloat16)
        s.scale = (0.5 + _rand(seed, 32, c["slots"])).tolist()
        s.y = torch.zeros(c["tokens"], c["rows"], device="cuda", dtype=DTYPES[c["y"]])
    else:
        s.ids = _ids(c, seed)
        s.offsets, s.order = _grouping(s.ids, c["groups"])
        s.cap = max(1, int((s.offsets[1:] - s.offsets[:-1]).max()))
        s.codes = _codes(c["kind"], c["group"], seed, 20, c["groups"], c["rows"], c["cols"])
        if op == "swiglu":
            s.up = _codes(c["kind"], c["group"], seed, 22, c["groups"], c["rows"], c["cols"])
        else:
            n_rows = c["tokens"] * c["per_row"]  # a down projection reads rows that are in their groups' order
        s.y = torch.zeros(c["tokens"] * c["per_row"], c["rows"], device="cuda", dtype=DTYPES[c["y"]])
    s.x = _randn(seed, 40, n_rows, c["cols"]).to(DTYPES[c["x"]])
    return s


# ---------------------------------------------------------------- the framework's handles

_CTX = None


def _ctx():
    global _CTX
    if _CTX is None:
        from hawking_amd import runtime
        _CTX = runtime.Context(0)
    return _CTX


def _vec(t):
    """A device tensor for the calls that take an object with a .ptr."""
    return SimpleNamespace(ptr=C.c_void_p(t.data_ptr()), t=t)


def _organs(p, c):
    from hawking_amd import organs as O
    ctx, rows, cols = _ctx(), c["rows"], c["cols"]
    if p.kind == "mixed":
        host = [[t.cpu().numpy().view("u2") if t.dtype == torch.float16 else t.cpu().numpy() for t in f]
                for f in (p.tags, p.bin_scales, p.bin_signs, p.q2_scales, p.q2_codes)]
        return [O.MixedPackedTensor(ctx, rows, cols, *f) for f in zip(*host)]
    s, q = p.scales.cpu().numpy().view("u2"), p.codes.cpu().numpy()
    if p.kind == "q4":
        return [O.Qwen80Q4PackedTensor(ctx, a, b, rows, cols, c["group"]) for a, b in zip(s, q)]
    make = {"q8": O.UniformFactorPacked, "bin": O.BinaryGroupPacked, "u3": O.UniformFactor3}[p.kind]
    return [make(ctx, a, b, rows, cols) for a, b in zip(s, q)]


def _rows(t, dtype):
    from hawking_amd import rows as R
    return R.Rows(_vec(t), t.shape[0], t.shape[1], dtype, t.stride(0))


def _bind(s):
    """What a program keeps: the organs, their sets, the adapters and the workspaces."""
    from hawking_amd import organs as O
    from hawking_amd import rows as R
    ctx, c = _ctx(), s.c
    if c["op"] == "group":
        n = s.ids.numel()
        s.out = {"offsets": torch.zeros(c["groups"] + 1, dtype=torch.int32, device="cuda"),
                 "order": torch.zeros(n, dtype=torch.int32, device="cuda"),
                 "pos": torch.zeros(n, dtype=torch.int32, device="cuda")}
        s.plan = R.RowGroups(ctx, n, c["groups"], **{k: _vec(v) for k, v in s.out.items()})
        s.ids_v = _vec(s.ids)
        return
    s.xr, s.yr = _rows(s.x, c["x"]), _rows(s.y, c["y"])
    if c["op"] == "combine":
        s.base_r = _rows(s.base, c["y"])
        s.pos_v, s.w_v = _vec(s.pos), _vec(s.w)
        return
    n_groups = c["slots"] if c["op"] == "lora" else c["groups"]
    s.plan = R.RowGroups(ctx, s.ids.numel(), n_groups, offsets=_vec(s.offsets), order=_vec(s.order))
    s.organs = _organs(_pack(c["kind"], *s.codes), c)
    if c["op"] == "lora":
        s.bank = R.LoraBank(ctx, s.organs[0], c["slots"], c["rank"])
        for i in range(c["slots"]):
            s.bank.set(i, c["rank"], _vec(s.a[i]), _vec(s.b[i]), "bf16", s.scale[i])
        s.gemm = R.LoraGemm(ctx, s.organs[0], s.bank, c["tokens"], c["x"], c["y"])
    elif c["op"] == "swiglu":
        s.up_organs = _organs(_pack(c["kind"], *s.up), c)
        s.gemm = R.GroupedSwiGlu(ctx, O.OrganSet(ctx, s.organs), O.OrganSet(ctx, s.up_organs), s.x.shape[0], c["x"], c["y"])
    else:
        s.gemm = R.GroupedGemm(ctx, O.OrganSet(ctx, s.organs), s.x.shape[0], c["x"], c["y"])
    s.codes = s.up = None  # the organs hold the weights from here on


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _bind(s)
    elif case["op"] in ("swiglu", "product", "lora"):
        s.w = _pack(case["kind"], *s.codes)
        if case["op"] == "swiglu":
            s.w_up = _pack(case["kind"], *s.up)
        s.codes = s.up = None
    return s


# ---------------------------------------------------------------- the plain forms

def _unpack(b, width, count):
    """`count` values of `width` bits, LSB first, from the bytes of every row of b."""
    bits = (b.unsqueeze(-1) >> torch.arange(8, device=b.device, dtype=torch.uint8)) & 1
    v = bits.reshape(b.shape[0], -1, width)[:, :count]
    return (v << torch.arange(width, device=b.device, dtype=torch.uint8)).sum(-1, dtype=torch.uint8)


def _decode(p, c):
    """The f32 weights [n, rows, cols] of packed matrices."""
    rows, cols, size = c["rows"], c["cols"], c["rows"] * c["cols"]
    if p.kind == "mixed":
        tag = torch.stack(p.tags)
        n, groups = tag.shape[0], size // 128
        coin = _unpack(tag, 1, groups).bool()
        w = torch.empty(n, groups, 2, 64, device=tag.device)
        signs = _unpack(torch.cat(p.bin_signs).view(1, -1), 1, 1 << 62).view(-1, 2, 64).float()
        w[coin] = (2 * signs - 1) * torch.cat(p.bin_scales).float().view(-1, 1, 1)
        codes = _unpack(torch.cat(p.q2_codes).view(1, -1), 2, 1 << 62).view(-1, 2, 64).float()
        w[~coin] = (codes - 1.5) * torch.cat(p.q2_scales).float().view(-1, 2, 1)
        return w.view(n, rows, cols)
    n = p.codes.shape[0]
    s = p.scales.float().unsqueeze(-1)
    if p.kind == "q4":
        q = torch.stack([p.codes & 15, p.codes >> 4], -1).view(n, s.shape[1], -1).float() - 8
    elif p.kind == "q8":
        q = p.codes.view(n, s.shape[1], -1).float() - 127
    elif p.kind == "bin":
        q = _unpack(p.codes, 1, size).view(n, s.shape[1], -1).float() * 2 - 1
    else:
        q = _unpack(p.codes, 3, s.shape[1] * 64).view(n, s.shape[1], -1).float() - 3
    return (q * s).view(n, -1)[:, :size].reshape(n, rows, cols)


def _padded(s, x_rows):
    """Each grouped row's group and place in it, and the rows as [groups, capacity, cols] (zeros past a group's end)."""
    c = s.c
    i = torch.arange(x_rows.shape[0], device="cuda", dtype=torch.int32)
    g = torch.searchsorted(s.offsets[1:].contiguous(), i, right=True)
    inside = (g < c["groups"]).unsqueeze(1)
    gc = g.clamp(max=c["groups"] - 1)
    slot = torch.where(inside[:, 0], i - s.offsets[gc], 0).long()
    # rows without a group go to a matrix of their own, which is not used
    xp = torch.zeros(c["groups"] + 1, s.cap, c["cols"], device="cuda")
    xp[g, slot] = x_rows
    return xp[:-1], gc, slot, inside


def _plain(s):
    c = s.c
    if c["op"] == "group":
        offsets, order = _grouping(s.ids, c["groups"])
        pos = torch.empty_like(order)
        pos[order.long()] = torch.arange(order.numel(), device="cuda", dtype=torch.int32)
        return {"offsets": offsets, "order": order,
                "pos": torch.where((s.ids >= 0) & (s.ids < c["groups"]), pos, -1)}
    dtype = DTYPES[c["y"]]
    if c["op"] == "combine":
        x = s.x.float()[s.pos.clamp(min=0).long()]
        w = torch.where(s.pos >= 0, s.w, 0.0)
        return (s.base.float() + (x * w.unsqueeze(-1)).sum(1)).to(dtype)
    if c["op"] == "lora":
        x = s.x.float()
        y = x @ _decode(s.w, c)[0].t()
        scale = torch.tensor(s.scale, device="cuda")
        mid = torch.matmul(x, s.a.float().transpose(1, 2))  # every adapter's A x, [slots, rows, rank]
        mine = (s.ids.unsqueeze(0) == torch.arange(c["slots"], device="cuda").unsqueeze(1)).unsqueeze(-1)
        mid = torch.where(mine, mid * scale.view(-1, 1, 1), 0.0)
        return (y + torch.matmul(mid, s.b.float().transpose(1, 2)).sum(0)).to(dtype)
    x = s.x.float()
    if c["op"] == "swiglu":
        x = x[(s.order // c["per_row"]).long()]
    xp, g, slot, inside = _padded(s, x)
    y = torch.bmm(xp, _decode(s.w, c).transpose(1, 2))[g, slot]
    if c["op"] == "swiglu":
        y = y / (1 + torch.exp(-y)) * torch.bmm(xp, _decode(s.w_up, c).transpose(1, 2))[g, slot]
    return torch.where(inside, y, 0.0).to(dtype)


def run(s):
    if not own:
        return _plain(s)
    op = s.c["op"]
    if op == "group":
        s.plan.build(s.ids_v)
        return s.out
    if op == "combine":
        from hawking_amd import rows as R
        R.combine_rows(_ctx(), s.xr, s.pos_v, s.w_v, s.c["per_row"], s.yr, base=s.base_r)
    elif op == "swiglu":
        s.gemm(s.xr, s.plan, s.yr, gather=True, per_row=s.c["per_row"])
    elif op == "product":
        s.gemm(s.xr, s.plan, s.yr)
    else:
        s.gemm(s.xr, s.plan, s.yr)
    return s.y


# ---------------------------------------------------------------- what a pass cannot do without

_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _weight_bytes(c):
    bits = {"q4": 4 + 16 / c["group"], "q8": 8.25, "u3": 3.25, "bin": 1.125, "mixed": 0.7 * 1.125 + 0.3 * 2.25}[c["kind"]]
    return c["rows"] * c["cols"] * bits / 8


def work(case):
    c, op = case, case["op"]
    if op == "group":
        n = c["tokens"] * c["per_row"]
        return {"bytes": 12 * n + 4 * (c["groups"] + 1), "flops": 0}
    n = c["tokens"] * c.get("per_row", 1)
    if op == "combine":
        y = c["tokens"] * c["cols"] * _SIZE[c["y"]]
        return {"bytes": n * (1 - c["absent"]) * c["cols"] * _SIZE[c["x"]] + 2 * y + 8 * n, "flops": 2 * n * c["cols"]}
    if op == "lora":
        used = c["slots"] * (1 - (1 - 1 / c["slots"]) ** c["requests"])
        io = n * (c["cols"] * _SIZE[c["x"]] + c["rows"] * _SIZE[c["y"]])
        return {"bytes": _weight_bytes(c) + used * c["rank"] * (c["rows"] + c["cols"]) * 2 + io,
                "flops": 2 * n * (c["rows"] * c["cols"] + c["rank"] * (c["rows"] + c["cols"]))}
    mats = 2 if op == "swiglu" else 1
    used = c["groups"] * (1 - (1 - 1 / c["groups"]) ** n)
    x_rows = c["tokens"] if op == "swiglu" else n
    return {"bytes": mats * used * _weight_bytes(c) + x_rows * c["cols"] * _SIZE[c["x"]] + n * c["rows"] * _SIZE[c["y"]],
            "flops": 2 * mats * n * c["rows"] * c["cols"]}


# ---------------------------------------------------------------- the definition, in 64 bits

def _value(kind, code, scale, coin, g, rows, cols):
    """Matrix g in f64, from its integer codes."""
    q = code[g].double()
    if kind == "mixed":
        binary = coin[g].repeat_interleave(128)
        q = torch.where(binary, 2 * q - 1, q - 1.5)
        unit = 64
    else:
        unit = {"bin": 128, "q8": 64, "u3": 64}.get(kind) or q.numel() // scale.shape[1]
        q = 2 * q - 1 if kind == "bin" else q - {"q4": 8, "q8": 127, "u3": 3}[kind]
    w = q * scale[g].double().repeat_interleave(unit)[: q.numel()]
    return w[: rows * cols].view(rows, cols)


def exact(case, seed):
    c, op = case, case["op"]
    if op == "group":
        return None  # whole numbers
    s = _inputs(c, seed)
    if op == "combine":
        y = s.base.double()
        for r in range(c["per_row"]):
            at = s.pos[:, r].long()
            live = at >= 0
            y[live] += s.w[live, r].double().unsqueeze(1) * s.x[at[live]].double()
        return y
    if op == "lora":
        w = _value(c["kind"], *s.codes, 0, c["rows"], c["cols"])
        y = torch.empty(c["tokens"], c["rows"], device="cuda", dtype=torch.float64)
        for a in [-1] + list(range(c["slots"])):
            at = (s.ids == a).nonzero()[:, 0]
            if not at.numel():
                continue
            x = s.x[at].double()
            y[at] = x @ w.t()
            if a >= 0:
                y[at] += s.scale[a] * ((x @ s.a[a].double().t()) @ s.b[a].double().t())
        return y
    n = c["tokens"] * c["per_row"]
    y = torch.zeros(n, c["rows"], device="cuda", dtype=torch.float64)
    edges = s.offsets.tolist()
    for g in range(c["groups"]):
        lo, hi = edges[g], edges[g + 1]
        if lo == hi:
            continue
        at = (s.order[lo:hi] // c["per_row"]).long() if op == "swiglu" else torch.arange(lo, hi, device="cuda")
        x = s.x[at].double()
        v = x @ _value(c["kind"], *s.codes, g, c["rows"], c["cols"]).t()
        if op == "swiglu":
            v = v * torch.sigmoid(v) * (x @ _value(c["kind"], *s.up, g, c["rows"], c["cols"]).t())
        y[lo:hi] = v
    return y
