"""What the 8-bit operators are measured on: products with weights in e4m3 and a scale for each block of 128, at the sizes of this engine's named models.

The arithmetic, the same in every form.  A row of activations is cut into blocks of 128 along K (the last one filled with zeros).  With a = max |x| of a block,
its scale s is the smallest power of two, 2^-100 at least, for which a <= 448 s (1 where the block is zero), and its codes are x / s rounded to e4m3; a block
that holds an infinity or a NaN has the scale NaN and codes of zero.  Weights are e4m3 codes with an fp32 scale t for each block of 128 x 128.  The product is

    y[m, n] = act(sum_b s[m, b] t[n / 128, b] sum_{k in b} x8[m, k] w8[n, k]  +  bias[n])

and a gated activation takes columns in runs of 32: 16 of the gate, then 16 of the branch that it multiplies.

Kinds of case (field ``kind``):
  rows     ``ops.fp8_rows``: rows to codes and scales, taken in order or through an index
  linear   ``ops.linear``: dense layers
  experts  ``ops.expert_linear``: rows sorted by expert, each run with its expert's matrix
  slots    ``ops.expert_gemv``: one row and one expert per slot, the step of a few tokens
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
ACTS = ("none", "swiglu", "swiglu_oai", "geglu")


# ------------------------------------------------------------------ the cases
def listed():
    linear = dict(kind="linear", act="none", bias=False, out="bf16")
    experts = dict(kind="experts", act="swiglu", bias=False, spread=0.5)
    slots = dict(kind="slots", bias=False)
    return [
        # the hidden state of one token, before the projections that share it
        dict(name="rows_token", kind="rows", rows=1, k=4096, index=False, dtype="bf16"),
        # what the down projection of a 4096-token prompt reads, Llama-3-8B
        dict(name="rows_prompt", kind="rows", rows=4096, k=14336, index=False, dtype="bf16"),
        # qkv projection of one token, Llama-3-8B
        dict(linear, name="linear_token", rows=1, n=6144, k=4096),
        # gate and up projection of a decode batch of eight, Llama-3-8B
        dict(linear, name="linear_gated_8", rows=8, n=28672, k=4096, act="swiglu"),
        # down projection of a decode batch of 40
        dict(linear, name="linear_batch_40", rows=40, n=4096, k=14336),
        # qkv projection of a short prompt, gpt-oss: K ends inside a block, rows inside a tile, results in 32 bits
        dict(linear, name="linear_ragged", rows=333, n=5120, k=2880, bias=True, out="fp32"),
        # output of the feed-forward for one chunk of a prompt, Llama-3-8B
        dict(linear, name="linear_chunk", rows=512, n=4096, k=14336),
        # gate and up projection of a 4096-token prompt, Llama-3-8B
        dict(linear, name="linear_prompt", rows=4096, n=28672, k=4096, act="swiglu"),
        # gate and up rows of 64 concurrent requests, Qwen3-MoE: a few rows for each of 128 experts
        dict(experts, name="experts_batch", tokens=64, n=1536, k=2048, experts=128, topk=8),
        # the same for a 2048-token prompt on experts of gpt-oss-20b's size, with biases
        dict(experts, name="experts_prompt", tokens=2048, n=5760, k=2880, experts=32, topk=4, act="swiglu_oai", bias=True),
        # one token, ten of 512 experts, Qwen3-Next-80B
        dict(slots, name="slots_token", tokens=1, n=1024, k=2048, experts=512, topk=10, act="swiglu", shared=True),
        # down projection of four tokens, eight of 128 experts, Qwen3-MoE: every slot has a row of its own
        dict(slots, name="slots_down_4", tokens=4, n=2048, k=768, experts=128, topk=8, act="none", shared=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows"] * 2 + ["linear"] * 5 + ["experts"] * 3 + ["slots"] * 2)
    odd = rng.random() < 0.4
    if kind == "rows":
        k = _log_int(rng, 64, 16384)
        k = k if odd else max(64, k // 64 * 64)
        return dict(kind=kind, rows=_log_int(rng, 1, min(8192, (58 << 20) // k)), k=k, index=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]))
    act = rng.choice(["none", "none", "swiglu", "swiglu_oai", "geglu"])
    if kind == "linear":
        n, k = rng.choice([(6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336), (5120, 2880), (2880, 4096), (12288, 2048), (2048, 8192)])
        if odd:
            n, k = _log_int(rng, 100, 20000), _log_int(rng, 100, 10000)
        if act != "none":
            n = n // 32 * 32
        return dict(kind=kind, rows=min(_log_int(rng, 1, 6000), int(4.8e11 / (n * k))), n=n, k=k, act=act, bias=rng.random() < 0.3, out=rng.choice(["bf16", "bf16", "fp32"]))
    n, k, experts, topk = rng.choice([(1536, 2048, 128, 8), (2048, 768, 128, 8), (1024, 2048, 512, 10), (2048, 512, 512, 10), (5760, 2880, 32, 4), (2880, 2880, 32, 4)])
    if odd:
        n, k = _log_int(rng, 100, 4000) // 32 * 32, _log_int(rng, 100, 3000)
        experts = rng.choice([3, 8, 17, 60])
        topk = min(topk, experts - 1)
    if kind == "experts":
        return dict(kind=kind, tokens=min(_log_int(rng, 5, 4096), int(4.8e11 / (n * k * topk))), n=n, k=k, experts=experts, topk=topk, act=act, bias=rng.random() < 0.3,
                    spread=rng.choice([0.0, 0.5, 1.0]))
    return dict(kind=kind, tokens=rng.randint(1, 8), n=n, k=k, experts=experts, topk=topk, act=act, bias=rng.random() < 0.3, shared=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _gen(seed, name):
    h = 14695981039346656037
    for ch in f"{seed}/{name}".encode():
        h = ((h ^ ch) * 1099511628211) & ((1 << 62) - 1)
    return torch.Generator(device=DEV).manual_seed(h)


def _activations(seed, rows, k, dtype=torch.bfloat16):
    """Rows of unit size as a norm leaves them: most channels small, a few large ones, the same in every row."""
    g = _gen(seed, "x")
    x = torch.randn(rows, k, generator=g, device=DEV)
    return (x * torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))).to(dtype)


def _weights(seed, experts, n, k):
    """Codes and scales as a checkpoint holds them: blocks of 128 x 128 scaled by their largest magnitude over 448."""
    g = _gen(seed, "w")
    codes = torch.empty(experts, n, k, device=DEV, dtype=torch.float8_e4m3fn)
    for e in range(experts):
        w = torch.randn(n, k, generator=g, device=DEV)
        codes[e] = (w.clamp_(-4.0, 4.0) * 112.0).to(torch.float8_e4m3fn)
    scales = (0.6 + 0.8 * torch.rand(experts, -(-n // BLOCK), -(-k // BLOCK), generator=g, device=DEV)) * (k ** -0.5 / 112.0)
    return codes, scales


def prepare(case, seed):
    kind, k = case["kind"], case["k"]
    if kind == "rows":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        x = _activations(seed, case["rows"], k, dtype)
        index = torch.randint(0, case["rows"], (case["rows"],), generator=_gen(seed, "index"), device=DEV, dtype=torch.int32) if case["index"] else None
        return dict(kind=kind, x=x, index=index)
    experts = case.get("experts", 1)
    codes, scales = _weights(seed, experts, case["n"], k)
    s = dict(kind=kind, codes=codes, scales=scales, act=case["act"], out_f32=case.get("out") == "fp32")
    s["bias"] = torch.randn(experts, case["n"], generator=_gen(seed, "bias"), device=DEV) if case["bias"] else None
    if kind == "linear":
        s["x"] = _activations(seed, case["rows"], k)
    else:
        tokens, topk = case["tokens"], case["topk"]
        g = _gen(seed, "route")
        logits = torch.randn(tokens, experts, generator=g, device=DEV) + case.get("spread", 0.0) * torch.randn(experts, generator=g, device=DEV)
        idx = logits.topk(topk, dim=1).indices.to(torch.int32)
        if kind == "slots":
            s.update(slot=idx.reshape(-1).contiguous(), x_div=topk if case["shared"] else 1)
            s["x"] = _activations(seed, tokens if case["shared"] else tokens * topk, k)
        else:
            s["x"] = _activations(seed, tokens, k)
            flat = idx.reshape(-1).long()
            order = torch.sort(flat, stable=True).indices
            counts = torch.bincount(flat, minlength=experts)
            first = torch.zeros(experts + 1, dtype=torch.long, device=DEV)
            first[1:] = counts.cumsum(0)
            s.update(order=order, expert=flat[order], counts=counts, first=first, token=(order // topk).to(torch.int32), most=int(counts.max()))
    if own:
        from machx_inference_engine_b200 import ops
        s["w"] = ops.from_fp8(codes, scales)
        s["act_id"] = {"none": ops.ACT_NONE, "swiglu": ops.ACT_SWIGLU, "swiglu_oai": ops.ACT_SWIGLU_OAI, "geglu": ops.ACT_GEGLU}[case["act"]]
        if kind == "experts":
            s["pk"] = ops.moe_pack(idx, experts, tile=1)
    return s


# ------------------------------------------------------------------ plain forms
def _quantise(x):
    """Codes [rows, blocks * 128] and scales [blocks, rows], fp32."""
    rows, k = x.shape
    blocks = -(-k // BLOCK)
    x = torch.nn.functional.pad(x.to(torch.float32), (0, blocks * BLOCK - k)).view(rows, blocks, BLOCK)
    top = x.abs().amax(dim=-1)
    finite = torch.isfinite(top)
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-100)
    e = torch.where((top > 0) & finite, e, torch.zeros_like(e))
    scale = ((e.to(torch.int32) + 127) << 23).view(torch.float32)       # 2^e, exactly
    codes = (torch.where(finite[..., None], x, torch.zeros_like(x)) / scale[..., None]).to(torch.float8_e4m3fn)
    scale = torch.where(finite, scale, torch.full_like(scale, math.nan))
    return codes.view(rows, blocks * BLOCK), scale.t().contiguous()


def _values(x):
    codes, scale = _quantise(x)
    return codes.to(torch.float32) * scale.t().repeat_interleave(BLOCK, dim=1)


def _decoded(codes, scales):
    """Weights [.., n, blocks * 128] in fp32."""
    n, k = codes.shape[-2:]
    blocks = scales.shape[-1]
    t = scales.repeat_interleave(BLOCK, dim=-2)[..., :n, :].repeat_interleave(BLOCK, dim=-1)
    w = torch.nn.functional.pad(codes.view(torch.uint8), (0, blocks * BLOCK - k)).view(torch.float8_e4m3fn)
    return w.to(torch.float32) * t


def _activate(y, act):
    if act == "none":
        return y
    v = y.unflatten(-1, (y.shape[-1] // 32, 2, 16))
    g, u = v[..., 0, :], v[..., 1, :]
    if act == "swiglu":
        r = g * torch.sigmoid(g) * u
    elif act == "swiglu_oai":
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        r = g * torch.sigmoid(1.702 * g) * (u + 1.0)
    else:
        r = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
    return r.flatten(-2)


def run(s):
    kind = s["kind"]
    if own:
        from machx_inference_engine_b200 import ops
        if kind == "rows":
            q = ops.fp8_rows(s["x"], index=s["index"])
            return q.codes, q.scale
        if kind == "linear":
            return ops.linear(s["x"], s["w"], bias=None if s["bias"] is None else s["bias"][0], act=s["act_id"], out_f32=s["out_f32"])
        if kind == "experts":
            return ops.expert_linear(s["x"], s["w"], s["pk"], x_index=s["pk"].packed_token, bias=s["bias"], act=s["act_id"])
        return ops.expert_gemv(s["x"], s["w"], s["slot"], x_div=s["x_div"], bias=s["bias"], act=s["act_id"])
    if kind == "rows":
        return _quantise(s["x"] if s["index"] is None else s["x"][s["index"].long()])
    x = _values(s["x"])
    if kind == "linear":
        y = x @ _decoded(s["codes"][0], s["scales"][0]).t()
        if s["bias"] is not None:
            y = y + s["bias"][0]
        y = _activate(y, s["act"])
        return y if s["out_f32"] else y.to(torch.bfloat16)
    if kind == "slots":
        e = s["slot"].long()
        x = x.repeat_interleave(s["x_div"], dim=0)
        y = torch.bmm(_decoded(s["codes"].view(torch.uint8)[e].view(torch.float8_e4m3fn), s["scales"][e]), x[..., None])[..., 0]
        if s["bias"] is not None:
            y = y + s["bias"][e]
        return _activate(y, s["act"]).to(torch.bfloat16)
    experts = s["codes"].shape[0]
    at = torch.arange(s["expert"].numel(), device=x.device) - s["first"][s["expert"]]
    padded = torch.zeros(experts, s["most"], x.shape[1], device=x.device)
    padded[s["expert"], at] = x[s["token"].long()]
    y = torch.bmm(padded, _decoded(s["codes"], s["scales"]).transpose(1, 2))[s["expert"], at]
    if s["bias"] is not None:
        y = y + s["bias"][s["expert"]]
    return _activate(y, s["act"]).to(torch.bfloat16)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, k = case["kind"], case["k"]
    blocks = -(-k // BLOCK)
    if kind == "rows":
        rows = case["rows"]
        return dict(bytes=rows * k * (2 if case["dtype"] == "bf16" else 4) + rows * blocks * (BLOCK + 4) + (4 * rows if case["index"] else 0), flops=3 * rows * k)
    n = case["n"]
    n_out = n // 2 if case["act"] != "none" else n
    matrix = n * k + 4 * -(-n // BLOCK) * blocks + (4 * n if case["bias"] else 0)
    if kind == "linear":
        rows, x_rows, matrices = case["rows"], case["rows"], 1
    else:
        rows = case["tokens"] * case["topk"]
        x_rows = rows if kind == "slots" and not case["shared"] else case["tokens"]
        matrices = case["experts"] * (1.0 - (1.0 - case["topk"] / case["experts"]) ** case["tokens"])      # (experts that some token takes, if all are equally likely)
    return dict(bytes=int(matrices * matrix) + 2 * x_rows * k + rows * n_out * (4 if case.get("out") == "fp32" else 2) + (0 if kind == "linear" else 4 * rows), flops=2 * rows * n * k)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(x):
    """Values of the codes [rows, blocks, 128] and scales [rows, blocks], from the definition."""
    rows, k = x.shape
    blocks = (k + BLOCK - 1) // BLOCK
    v = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :k] = x.double()
    v = v.reshape(rows, blocks, BLOCK)
    a = v.abs().max(dim=2).values
    s = torch.full_like(a, 2.0 ** -100)
    for _ in range(230):                                     # doubled until it holds the block's largest
        s = torch.where(a > 448.0 * s, 2.0 * s, s)
    s = torch.where(a == 0, torch.ones_like(s), s)
    z = v / s[..., None]
    unit = torch.full_like(z, 2.0 ** -9)                     # steps of e4m3: eight of them in every octave from 2^-6 on
    for _ in range(15):
        unit = torch.where(z.abs() >= 16 * unit, 2 * unit, unit)
    return torch.round(z / unit) * unit, s


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"]
    if case["kind"] == "rows":
        if s["index"] is not None:
            x = x[s["index"].long()]
        q, scale = _exact_rows(x)
        return q.flatten(1), scale.t().contiguous()
    q, scale = _exact_rows(x)
    xv = (q * scale[..., None]).flatten(1)[:, :case["k"]]

    def product(rows, e):
        w = s["codes"][e].double()
        for b in range(s["scales"].shape[2]):
            w[:, b * BLOCK:(b + 1) * BLOCK] *= s["scales"][e][:, b].double().repeat_interleave(BLOCK)[:w.shape[0], None]
        y = rows @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"][e].double()
        if case["act"] == "none":
            return y
        columns = torch.arange(y.shape[1], device=y.device)
        gate, up = y[:, columns % 32 < 16], y[:, columns % 32 >= 16]
        if case["act"] == "swiglu":
            return gate / (1.0 + torch.exp(-gate)) * up
        if case["act"] == "swiglu_oai":
            gate = torch.minimum(gate, torch.full_like(gate, 7.0))
            up = torch.minimum(torch.maximum(up, torch.full_like(up, -7.0)), torch.full_like(up, 7.0))
            return gate / (1.0 + torch.exp(-1.702 * gate)) * (up + 1.0)
        return gate * 0.5 * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (gate + 0.044715 * gate ** 3))) * up

    if case["kind"] == "linear":
        return product(xv, 0)
    if case["kind"] == "slots":
        return torch.cat([product(xv[i // s["x_div"]][None], e) for i, e in enumerate(s["slot"].tolist())])
    counts, tokens = s["counts"].tolist(), s["token"].long()
    done, parts = 0, []
    for e, c in enumerate(counts):
        if c:
            parts.append(product(xv[tokens[done:done + c]], e))
            done += c
    return torch.cat(parts)
