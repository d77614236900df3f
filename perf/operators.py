"""Cases of the operators that train and serve transformer towers through 8-bit activations: the checkpoint of an
activation in 8 bits and its use in the backward pass, the root-mean-square norm with the residual's addition (16-bit
or e4m3 output), and the scaled embedding lookup with its gradient by tokens.

`run` computes each in its plain form (32-bit torch, rounded once at the end) unless `own` is set; then it makes the
calls of bifold_amd.hip.ops.  `exact` computes the same from the definitions in 64 bits.

The 8-bit checkpoint: a row is cut into groups of 32 columns (the last may be shorter).  A group has one exponent e, the
smallest for which round(max |x| 2^-e) <= 127, at least -126; its values are q = round(x 2^-e), ties to even, and read
back as q 2^e.  A group that holds an infinity or a NaN reads back as NaN.
"""
import math

import torch

own = False

GROUP = 32
EPS = 1e-6
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one MLP of ViT-L/14 at 336 pixels (577 tokens, width 4096), a training step of 64 images: the largest
        dict(name="gelu_vitl", op="gelu", rows=64 * 577, cols=4096, dtype="fp16", act="quick", strided=False),
        # one MLP of the CLIP text tower (77 tokens, width 2048) at 128 instructions
        dict(name="gelu_text", op="gelu", rows=128 * 77, cols=2048, dtype="bf16", act="tanh", strided=False),
        # exact mode on an odd width, one instruction
        dict(name="gelu_odd", op="gelu", rows=77, cols=1021, dtype="fp32", act="erf", strided=False),
        # the fp32 stream of a SigLIP tower (576 tokens, width 768) kept in 8 bits and read back: 128 images
        dict(name="stream_siglip", op="trip", rows=128 * 576, cols=768, dtype="fp32", strided=False),
        # fusion-stack rows read out of a wider buffer (the value columns of a packed projection)
        dict(name="stream_columns", op="trip", rows=5 * 275, cols=520, dtype="bf16", strided=True),
        # the norm in front of an e4m3 in-projection: ViT-B/16 (197 tokens, width 768) at 256 images
        dict(name="norm8_vitb", op="norm8", rows=256 * 197, cols=768, dtype="fp32", delta="fp16", strided=False),
        # a single token of a wide model, on its way to an e4m3 product
        dict(name="norm8_token", op="norm8", rows=1, cols=4096, dtype="bf16", delta="bf16", strided=False),
        # forward and backward of a norm whose stream is kept in 8 bits: ViT-L/14 at 64 images
        dict(name="norm_step_vitl", op="norm_step", rows=64 * 577, cols=1024, dtype="fp32", delta="fp16", strided=False),
        # the same at an odd width
        dict(name="norm_step_odd", op="norm_step", rows=1100, cols=1155, dtype="bf16", delta="bf16", strided=False),
        # token embeddings of 128 instructions padded to 64 tokens (SigLIP's vocabulary) and their gradient
        dict(name="embed_siglip", op="embed", tokens=128 * 64, cols=768, vocab=32000, dtype="fp16", context=64, pad=False),
        # one instruction of CLIP's vocabulary: the gradient is one write of the table's size
        dict(name="embed_one", op="embed", tokens=77, cols=512, vocab=49408, dtype="fp32", context=77, pad=False),
        # a language model's batch: long sequences, the padding's rows left out
        dict(name="embed_batch", op="embed", tokens=131072, cols=1024, vocab=65536, dtype="bf16", context=2048, pad=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["gelu", "trip", "norm8", "norm", "norm_step", "embed"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "embed":
        context = _log(rng, 8, 2048)
        return dict(op=op, tokens=min(131072, context * _log(rng, 1, 256)), cols=_log(rng, 32, 1024),
                    vocab=_log(rng, 256, 65536), dtype=dtype, context=context, pad=rng.random() < 0.5)
    cols = _log(rng, 16, 8192)
    if rng.random() < 0.5:
        cols = -(-cols // 32) * 32
    rows = _log(rng, 1, max(2, min(40000, 40_000_000 // cols)))
    case = dict(op=op, rows=rows, cols=cols, dtype=dtype, strided=rng.random() < 0.3)
    if op == "gelu":
        case["act"] = rng.choice(["quick", "erf", "tanh"])
    if op in ("norm8", "norm", "norm_step"):
        case["delta"] = rng.choice(["none", "bf16", "fp16"] if dtype == "fp32" else ["none", dtype])
    return case


# ------------------------------------------------------------------ inputs
def _rows(case, g, spread, mean=0.0):
    """[rows, cols] activations: normal values, some columns several times the others' size; a view of a wider
    buffer where the case is strided."""
    wide = case["cols"] + (24 if case["strided"] else 0)
    size = torch.rand(wide, generator=g, device="cuda").pow(8).mul(8).add(1).mul(spread)
    x = torch.randn(case["rows"], wide, generator=g, device="cuda").mul_(size).add_(mean).to(DTYPES[case["dtype"]])
    return x[:, 8:8 + case["cols"]] if case["strided"] else x


def _half(case):
    """The 16-bit type of the branch next to this stream (a 16-bit stream's own)."""
    return case["dtype"] if case["dtype"] != "fp32" else "fp16" if case.get("delta") == "none" else case["delta"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "embed":
        n, vocab, context = case["tokens"], case["vocab"], case["context"]
        # word frequencies fall like 1 / rank; the tail of each sequence is padding (token 1)
        ids = torch.rand(n, generator=g, device="cuda").mul_(math.log(vocab)).exp_().sub_(1).long().clamp_(0, vocab - 1)
        where = torch.arange(n, device="cuda")
        length = torch.randint(1, context + 1, (n // context + 1,), generator=g, device="cuda")
        ids = torch.where(where % context >= length[where // context], torch.ones_like(ids), ids)
        s["ids"] = ids.to(torch.int32).view(1, n)
        s["table"] = torch.randn(vocab, case["cols"], generator=g, device="cuda").mul_(0.02).to(DTYPES[case["dtype"]])
        s["dy"] = torch.randn(n, case["cols"], generator=g, device="cuda").mul_(0.05).to(DTYPES[case["dtype"]])
        s["scale"] = math.sqrt(case["cols"])
        s["flag"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return s
    if case["op"] == "gelu":
        s["pre"] = _rows(case, g, 0.6, -0.2)
        s["dy"] = _rows(case, g, 0.05)
        return s
    s["x"] = _rows(case, g, 1.0)
    if case["op"] == "trip":
        return s
    s["gamma"] = torch.randn(case["cols"], generator=g, device="cuda").mul_(0.1).add_(1)
    if case["delta"] != "none":
        s["delta"] = _rows(dict(case, dtype=case["delta"]), g, 0.5)
    if case["op"] == "norm_step":
        s["dy"] = torch.randn(case["rows"], case["cols"], generator=g, device="cuda").mul_(0.05).to(DTYPES[_half(case)])
        s["dres"] = torch.randn(case["rows"], case["cols"], generator=g, device="cuda").mul_(0.05).to(DTYPES[_half(case)])
    return s


# ------------------------------------------------------------------ plain forms
def _groups(x):
    """[rows, cols] as [rows, groups, 32], the last group filled up with zeros."""
    rows, cols = x.shape
    many = -(-cols // GROUP)
    full = x if many * GROUP == cols else torch.cat([x, x.new_zeros(rows, many * GROUP - cols)], 1)
    return full.reshape(rows, many, GROUP)


def _kept(x):
    """What the 8-bit checkpoint of a 32-bit tensor reads back as.  A group's exponent comes from the bits of its largest
    magnitude: its field less 6, and one more where the 7-bit value would round up to 128."""
    g = _groups(x)
    bits = g.abs().amax(2, keepdim=True).view(torch.int32)
    whole = bits < 0x7F800000
    code = torch.where(whole, (((bits + 0x10000) >> 23) - 6).clamp(min=1), 255)
    q = torch.where(whole, torch.round(g * ((254 - code).clamp(min=0) << 23).view(torch.float32)), 0.0)
    return (q * (code << 23).view(torch.float32)).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _inner(x):
    return 0.7978845608028654 * (x + 0.044715 * x * x * x)


def _act(x, act):
    if act == "quick":
        return x / (1 + torch.exp(-1.702 * x))
    if act == "erf":
        return 0.5 * x * torch.erfc(-0.7071067811865476 * x)
    return x / (1 + torch.exp(-2 * _inner(x)))


def _act_slope(x, act):
    if act == "erf":
        return 0.5 * torch.erfc(-0.7071067811865476 * x) + x * 0.3989422804014327 * torch.exp(-0.5 * x * x)
    if act == "quick":
        u, du = 1.702 * x, 1.702
    else:
        u, du = 2 * _inner(x), 2 * 0.7978845608028654 * (1 + 3 * 0.044715 * x * x)
    up = 1 / (1 + torch.exp(-u))
    return up + x * du * up / (1 + torch.exp(u))


def _norm(s, x):
    """(sum, 1 / rms, normed) in 32 bits."""
    x = x.float() + s["delta"].float() if "delta" in s else x.float()
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    return x, r, x * r * s["gamma"]


def _plain(s):
    case = s["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "gelu":
        pre = s["pre"].float()
        slope = _act_slope(_kept(pre), case["act"])
        return _act(pre, case["act"]).to(dtype), (s["dy"].float() * slope).to(dtype)
    if case["op"] == "trip":
        return _kept(s["x"].float()).to(dtype)
    if case["op"] == "embed":
        ids = s["ids"].view(-1).long()
        out = (s["table"][ids].float() * s["scale"]).to(dtype)
        live = s["dy"].double() * (ids != 1).unsqueeze(1) if case["pad"] else s["dy"].double()    # long sums: 64 bits
        grad = live.new_zeros(case["vocab"], case["cols"]).index_add_(0, ids, live)
        return out, (grad * s["scale"]).float()
    x, r, y = _norm(s, s["x"])
    if case["op"] == "norm":
        return y.to(DTYPES[_half(case)]), x.to(dtype)
    if case["op"] == "norm8":
        top = y.abs().amax(1)
        scale = torch.where(top > 0, top / 448, 1.0)
        return (y / scale.unsqueeze(1)).clamp(-448, 448).to(torch.float8_e4m3fn), scale, x.to(dtype)
    kept = _kept(x) * r
    dy = s["dy"].float()
    back = dy * s["gamma"]
    dx = r * (back - kept * (back * kept).mean(1, keepdim=True)) + s["dres"].float()
    return y.to(DTYPES[_half(case)]), x.to(dtype), dx.to(DTYPES[_half(case)]), (dy * kept).sum(0)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from bifold_amd.hip import lib as L
    from bifold_amd.hip import ops

    case = s["case"]
    if case["op"] == "gelu":
        act = {"quick": L.ACT_QUICK_GELU, "erf": L.ACT_ERF_GELU, "tanh": L.ACT_TANH_GELU}[case["act"]]
        y, kept = ops.act8_gelu_fwd(s["pre"], act)
        return y, ops.act8_gelu_bwd(s["dy"], kept, act)
    if case["op"] == "trip":
        kept = ops.act8_pack(s["x"])
        return ops.act8_unpack(kept, s["x"].dtype)
    if case["op"] == "embed":
        out = ops.embed_scaled_fwd(s["ids"], s["table"], s["scale"], s["flag"], s["table"].dtype)
        grad = ops.embed_scaled_bwd(s["dy"], s["ids"], case["vocab"], s["scale"], s["flag"],
                                    padding_idx=1 if case["pad"] else None)
        return out, grad
    x, delta = s["x"], s.get("delta")
    total = x if delta is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if case["op"] == "norm":
        y, _, _ = ops.rmsnorm_fwd(x, s["gamma"], DTYPES[_half(case)], delta=delta, x_out=total, eps=EPS)
        return y, total
    if case["op"] == "norm8":
        y, scale, _, _ = ops.rmsnorm_fwd_fp8(x, s["gamma"], delta=delta, x_out=total, eps=EPS)
        return y.view(torch.float8_e4m3fn), scale, total
    y, rstd, kept = ops.rmsnorm_fwd(x, s["gamma"], DTYPES[_half(case)], delta=delta, x_out=total, eps=EPS,
                                    save_stats=True, checkpoint=True)
    dgamma = torch.empty(case["cols"], dtype=torch.float32, device=x.device)
    dx = ops.rmsnorm_bwd(s["dy"], kept, s["gamma"], rstd, dgamma, dres=s["dres"])
    return y, total, dx, dgamma


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the least each pass reads, writes and computes
def work(case):
    if case["op"] == "embed":
        n, cols, size = case["tokens"], case["cols"], SIZES[case["dtype"]]
        return {"bytes": n * cols * 3 * size + 4 * n + 4 * case["vocab"] * cols, "flops": 3 * n * cols}
    many, size = case["rows"] * case["cols"], SIZES[case["dtype"]]
    kept = many + case["rows"] * -(-case["cols"] // GROUP)
    if case["op"] == "gelu":                  # read pre, dy; write y, dx; the checkpoint once each way
        return {"bytes": 4 * size * many + 2 * kept, "flops": 30 * many}
    if case["op"] == "trip":
        return {"bytes": 2 * size * many + 2 * kept, "flops": 4 * many}
    half = 2
    branch = 0 if case["delta"] == "none" else half + size          # read the branch, write the sum
    if case["op"] == "norm":
        return {"bytes": (size + branch + half) * many, "flops": 5 * many}
    if case["op"] == "norm8":
        return {"bytes": (size + branch + 1) * many + 4 * case["rows"], "flops": 7 * many}
    return {"bytes": (size + branch + half + 3 * half) * many + 2 * kept, "flops": 18 * many}


# ------------------------------------------------------------------ the definitions in 64 bits
def _kept64(x):
    rows, cols = x.shape
    out = torch.empty(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device).zero_()
    out[:, :cols] = x
    out = out.unflatten(1, (-1, 32))
    fraction, power = torch.frexp(out.abs().max(2, keepdim=True).values)     # fraction 2^power, fraction in [1/2, 1)
    power = power - 7 + (fraction * 128 >= 127.5)
    power = torch.where(fraction == 0, -126, power.clamp(min=-126))
    step = ((power.long() + 1023) << 52).view(torch.float64)                 # 2^power, without pow's rounding
    return ((out / step).round() * step).flatten(1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        ids = s["ids"][0].long()
        out = s["table"].double().index_select(0, ids) * s["scale"]
        weights = s["dy"].double() * s["scale"]
        if case["pad"]:
            weights[ids == 1] = 0
        grad = torch.zeros(case["vocab"], case["cols"], dtype=torch.float64, device="cuda")
        grad.scatter_add_(0, ids[:, None].expand_as(weights), weights)
        return out, grad
    if case["op"] == "trip":
        return _kept64(s["x"].double())
    if case["op"] == "gelu":
        pre, at, dy = s["pre"].double(), _kept64(s["pre"].double()), s["dy"].double()
        if case["act"] == "erf":
            half = torch.special.ndtr
            return pre * half(pre), dy * (half(at) + at * torch.exp(-at * at / 2) / math.sqrt(2 * math.pi))
        if case["act"] == "quick":
            gate = torch.sigmoid(1.702 * at)
            return pre * torch.sigmoid(1.702 * pre), dy * gate * (1 + 1.702 * at * (1 - gate))
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (at + 0.044715 * at ** 3))
        y = pre * torch.sigmoid(2 * c * (pre + 0.044715 * pre ** 3))
        return y, dy * (0.5 * (1 + t) + 0.5 * at * (1 - t * t) * c * (1 + 0.134145 * at ** 2))
    x = s["x"].double()
    if "delta" in s:
        x = x + s["delta"].double()
    rms = x.pow(2).mean(1, keepdim=True).add(EPS).sqrt()
    y = x / rms * s["gamma"].double()
    if case["op"] == "norm":
        return y, x
    if case["op"] == "norm8":
        top = y.abs().max(1).values
        scale = torch.where(top == 0, torch.ones_like(top), top / 448)
        return y / scale[:, None], scale, x
    hat = _kept64(x.float().double()) / rms          # the checkpoint is taken of the 32-bit sum
    up = s["dy"].double() * s["gamma"].double()
    dx = (up - hat * (up * hat).sum(1, keepdim=True) / case["cols"]) / rms + s["dres"].double()
    return y, x, dx, (s["dy"].double() * hat).sum(0)
