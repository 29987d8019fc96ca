"""Cases of the 4-bit group-quantized operators and of the logits step, for timing and comparison.

Four operators: `quantize` (fp32 / bf16 weights to 4-bit codes with one bf16 scale per group, and
back to values), `embed` (rows of a 4-bit table), `linear` (tokens times 4-bit weights) and `logits`
(penalties, biases, allowed-token mask, greedy token).  `run` computes a case in elementary torch
operations, or with `own` set by the calls that a program makes of vvllm_b200.

The format: row n of `codes` (uint8) holds element 2j in the low and 2j+1 in the high four bits of
byte j, as q + 8 with q in -8..7; w[n, k] = q * scales[n, k // group], scales in bf16.
"""
import torch

own = False

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # a whole checkpoint's small MLP projection, as stored (bf16), quantized at load
        dict(name="quantize bf16 4864x896", op="quantize", n=4864, k=896, group=64, src="bf16"),
        # a large projection from fp32 weights: the longest part of quantizing a 7B model
        dict(name="quantize fp32 18944x3584", op="quantize", n=18944, k=3584, group=128, src="fp32"),
        # the token lookup of one decode step in a tied, 4-bit table: launch latency
        dict(name="embed 1 of 151936x896", op="embed", r=1, n=151936, k=896, group=64, out="fp16"),
        # the lookup of a long prompt
        dict(name="embed 2048 of 152064x3584", op="embed", r=2048, n=152064, k=3584, group=128, out="fp32"),
        # a small model's attention projection, one token: launch latency
        dict(name="linear 1x896x896", op="linear", m=1, n=896, k=896, group=64, x="fp16", out="fp16", bias=True,
             residual=False),
        # gate and up of a 7B decode step
        dict(name="linear 1x37888x3584", op="linear", m=1, n=37888, k=3584, group=128, x="fp16", out="fp16",
             bias=False, residual=False),
        # its down projection with fp32 activations, fine groups and the residual connection
        dict(name="linear 1x3584x18944 fp32", op="linear", m=1, n=3584, k=18944, group=32, x="fp32", out="fp32",
             bias=False, residual=True),
        # the output head for eight sequences, logits in fp32
        dict(name="linear 8x152064x3584", op="linear", m=8, n=152064, k=3584, group=128, x="fp16", out="fp32",
             bias=False, residual=False),
        # prefill of a prompt through the down projection
        dict(name="linear 512x3584x18944", op="linear", m=512, n=3584, k=18944, group=128, x="fp16", out="fp16",
             bias=True, residual=False),
        # one sequence's decode step: every penalty, a short history, no mask
        dict(name="logits 1x151936", op="logits", m=1, v=151936, hist=200, biases=0, mask=False, empty=False,
             x="fp16", out="fp16"),
        # a small vocabulary of odd size: rows that start unaligned, biases, a grammar mask
        dict(name="logits 7x32001", op="logits", m=7, v=32001, hist=1000, biases=300, mask=True, empty=True,
             x="fp16", out="fp32"),
        # a full batch with long histories under a grammar
        dict(name="logits 64x152064", op="logits", m=64, v=152064, hist=4096, biases=0, mask=True, empty=False,
             x="fp32", out="fp32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(lo * (hi / lo) ** rng.random() + 0.5)))


def _k(rng, lo, hi):
    """A row length: mostly whole groups as models have them, some whole 32s, some anything."""
    k, p = _log(rng, lo, hi), rng.random()
    if p < 0.6:
        return min(hi, max(128, k // 128 * 128))
    return max(32, k // 32 * 32) if p < 0.8 else k


def draw(rng):
    p, group = rng.random(), rng.choice((32, 64, 128))
    if p < 0.15:
        k = _k(rng, 32, 18944)
        n = min(_log(rng, 16, 37888), 18944 * 3584 // k)
        return dict(op="quantize", n=n, k=k, group=group, src=rng.choice(("bf16", "fp32")))
    if p < 0.3:
        k, n = _k(rng, 32, 3584), _log(rng, 1000, 152064)
        return dict(op="embed", r=_log(rng, 1, 2048), n=n, k=k, group=group, out=rng.choice(("fp16", "fp32")))
    if p < 0.75:
        k = _k(rng, 32, 18944)
        n = _log(rng, 16, 152064)
        n = min(n // 64 * 64 if n >= 64 and rng.random() < 0.5 else n, 152064 * 3584 // k)
        m = _log(rng, 1, 512)
        m = max(1, min(m, 512 * 3584 * 18944 // (n * k)))
        return dict(op="linear", m=m, n=n, k=k, group=group, x=rng.choice(("fp16", "fp16", "fp32")),
                    out=rng.choice(("fp16", "fp32")), bias=rng.random() < 0.5, residual=rng.random() < 0.4)
    m, v = _log(rng, 1, 64), _log(rng, 1000, 152064)
    return dict(op="logits", m=m, v=v, hist=_log(rng, 1, 4096), biases=rng.choice((0, 0, 20, 300)),
                mask=rng.random() < 0.5, empty=m > 1 and rng.random() < 0.3, x=rng.choice(("fp16", "fp32")),
                out=rng.choice(("fp16", "fp32")))


def work(case):
    c = dict(case)
    if c["op"] == "logits":
        out = SIZE[c["out"]] + SIZE[c["x"]] + (1 / 8 if c["mask"] else 0)
        return {"bytes": c["m"] * (c["v"] * out + 4 * c["hist"] + 8 * c["biases"] + 24), "flops": 6 * c["m"] * c["v"]}
    n, k = c["n"], c["k"]
    row = (k + 1) // 2 + 2 * -(-k // c["group"])  # a row's codes and scales
    if c["op"] == "quantize":
        return {"bytes": n * (k * (SIZE[c["src"]] + 4) + 2 * -(-k // c["group"])), "flops": 3 * n * k}
    if c["op"] == "embed":
        return {"bytes": c["r"] * (4 + row + k * SIZE[c["out"]]), "flops": c["r"] * k}
    m = c["m"]
    out = SIZE[c["out"]] * (2 if c["residual"] else 1)
    return {"bytes": n * row + m * k * SIZE[c["x"]] + m * n * out + (4 * n if c["bias"] else 0), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------ inputs

def _packed(g, n, k, group):
    """Codes and scales as quantizing normal weights of deviation 0.02 leaves them: the codes'
    distribution is a rounded normal whose largest value in a group is near 7."""
    ng = -(-k // group)
    spread = 7 / {32: 2.1, 64: 2.4, 128: 2.65}[group]  # the mean largest |value| of a group, in deviations
    codes = torch.empty((n, (k + 1) // 2), dtype=torch.uint8, device="cuda")
    for i in range(0, n, 16384):  # bounds what the normal values take
        z = torch.randn((min(16384, n - i), 2 * codes.shape[1]), generator=g, device="cuda").mul_(spread)
        q = z.round_().clamp_(-7, 7).add_(8).to(torch.uint8)
        if k % 2:
            q[:, k] = 8
        codes[i:i + 16384] = q[:, 0::2] | (q[:, 1::2] << 4)
    scales = (0.02 / spread) * (0.8 + 0.4 * torch.rand((n, ng), generator=g, device="cuda"))
    return codes, scales.to(torch.bfloat16)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "logits":
        m, v, h, b = c["m"], c["v"], c["hist"], c["biases"]
        s["logits"] = (4 * torch.randn((m, v), generator=g, device="cuda")).to(DT[c["x"]])
        # tokens repeat: a text draws most of its tokens from a few thousand
        s["history"] = (v * torch.rand((m, h), generator=g, device="cuda") ** 3).to(torch.int32).clamp_(max=v - 1)
        s["history_len"] = torch.randint(h // 2, h + 1, (m,), generator=g, device="cuda", dtype=torch.int32)
        s["prompt_len"] = s["history_len"] // 3
        s["repetition"] = 1 + 0.5 * torch.rand((m,), generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand((m,), generator=g, device="cuda")
        s["frequency"] = 0.3 * torch.rand((m,), generator=g, device="cuda")
        s["bias_ids"] = s["bias_values"] = s["bias_len"] = s["allowed"] = None
        if b:
            s["bias_ids"] = torch.randint(0, v, (m, b), generator=g, device="cuda", dtype=torch.int32)
            s["bias_values"] = 3 * torch.randn((m, b), generator=g, device="cuda")
            s["bias_len"] = torch.randint(0, b + 1, (m,), generator=g, device="cuda", dtype=torch.int32)
        if c["mask"]:  # a grammar allows a run of tokens here and there
            s["allowed"] = torch.randint(-2**31, 2**31, (m, (v + 31) // 32), generator=g, device="cuda").to(torch.int32)
            s["allowed"] &= -(torch.rand(s["allowed"].shape, generator=g, device="cuda") < 0.2).to(torch.int32)
            if c["empty"]:
                s["allowed"][-1] = 0
        s["out"] = torch.empty((m, v), dtype=DT[c["out"]], device="cuda")
        s["token"] = torch.empty((m,), dtype=torch.int32, device="cuda")
        return s
    n, k, group = c["n"], c["k"], c["group"]
    if c["op"] == "quantize":
        s["w"] = (0.02 * torch.randn((n, k), generator=g, device="cuda")).to(DT[c["src"]])
        s["codes"] = torch.empty((n, (k + 1) // 2), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty((n, -(-k // group)), dtype=torch.bfloat16, device="cuda")
        s["out"] = torch.empty((n, k), dtype=torch.float32, device="cuda")
        return s
    s["codes"], s["scales"] = _packed(g, n, k, group)
    if c["op"] == "embed":
        s["rows"] = torch.randint(0, n, (c["r"],), generator=g, device="cuda", dtype=torch.int32)
        s["out"] = torch.empty((c["r"], k), dtype=DT[c["out"]], device="cuda")
        return s
    m = c["m"]
    s["x"] = torch.randn((m, k), generator=g, device="cuda").to(DT[c["x"]])
    s["bias"] = 0.1 * torch.randn((n,), generator=g, device="cuda") if c["bias"] else None
    s["residual"] = torch.randn((m, n), generator=g, device="cuda").to(DT[c["out"]]) if c["residual"] else None
    s["out"] = torch.empty((m, n), dtype=DT[c["out"]], device="cuda")
    return s


# ------------------------------------------------------------------------------------------ passes

def run(state):
    op = state["case"]["op"]
    if own:
        return {"quantize": _own_quantize, "embed": _own_embed, "linear": _own_linear, "logits": _own_logits}[op](state)
    return {"quantize": _quantize, "embed": _embed, "linear": _linear, "logits": _logits}[op](state)


def _own_quantize(s):
    import vvllm_b200 as v

    if s["w"].dtype == torch.bfloat16:
        v.quantize_q4_bf16(s["w"], s["codes"], s["scales"], s["case"]["group"])
    else:
        v.quantize_q4(s["w"], s["codes"], s["scales"], s["case"]["group"])
    v.dequantize_q4(s["out"], s["codes"], s["scales"], s["case"]["group"])
    return {"values": s["out"], "scales": s["scales"]}


def _own_embed(s):
    import vvllm_b200 as v

    v.dequantize_q4(s["out"], s["codes"], s["scales"], s["case"]["group"], rows=s["rows"])
    return s["out"]


def _own_linear(s):
    import vvllm_b200 as v

    if s["residual"] is None:
        v.linear_q4(s["out"], s["x"], s["codes"], s["scales"], s["case"]["group"], s["bias"])
    else:
        v.linear_q4_add(s["out"], s["x"], s["codes"], s["scales"], s["case"]["group"], s["bias"], s["residual"])
    return s["out"]


def _own_logits(s):
    import vvllm_b200 as v

    v.process_logits(s["out"], s["logits"], s["token"], history=s["history"], history_len=s["history_len"],
                     prompt_len=s["prompt_len"], repetition=s["repetition"], presence=s["presence"],
                     frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                     bias_len=s["bias_len"], allowed=s["allowed"])
    return {"logits": s["out"], "token": s["token"]}


def _values(codes, scales, k, group):
    """fp32 [rows, k] of 4-bit rows; exact, a 4-bit integer times an 8-bit significand."""
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1)[:, :k].float() - 8
    s = scales.float()
    if k % group:
        return q * s.repeat_interleave(group, dim=1)[:, :k]
    return (q.view(len(q), -1, group) * s.unsqueeze(-1)).view(len(q), k)


def _quantize(s):
    w, group = s["w"].float(), s["case"]["group"]
    n, k = w.shape
    pad = -k % group
    if pad:
        w = torch.cat((w, w.new_zeros((n, pad))), dim=1)
    w = w.view(n, -1, group)
    top = w.abs().amax(dim=-1)
    scale = (top / torch.full_like(top, 7)).to(torch.bfloat16)  # a division: by a number it would be a product
    f = scale.float().unsqueeze(-1)
    q = torch.where(f > 0, torch.round(w / f), 0.0).clamp(-8, 7)  # round: ties to even
    return {"values": (q * f).view(n, -1)[:, :k].contiguous(), "scales": scale}


def _embed(s):
    rows = s["rows"].long()
    return _values(s["codes"][rows], s["scales"][rows], s["case"]["k"], s["case"]["group"]).to(s["out"].dtype)


def _linear(s):
    y = s["x"].float() @ _values(s["codes"], s["scales"], s["case"]["k"], s["case"]["group"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out"].dtype)


def _logits(s):
    x, hist = s["logits"].float(), s["history"].long()
    m, v = x.shape
    at = torch.arange(hist.shape[1], device="cuda")
    live = at < s["history_len"].unsqueeze(1)
    made = live & (at >= s["prompt_len"].unsqueeze(1))
    zero = torch.zeros((m, v), dtype=torch.int64, device="cuda")
    seen = zero.scatter_add(1, hist, live.long()) > 0
    count = zero.scatter_add(1, hist, made.long())
    rep = s["repetition"].unsqueeze(1)
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, x - s["frequency"].unsqueeze(1) * count.float(), x)
    x = torch.where(count > 0, x - s["presence"].unsqueeze(1), x)
    if s["bias_ids"] is not None:  # a token listed twice takes its last bias
        at = torch.arange(s["bias_ids"].shape[1], device="cuda")
        entry = torch.where(at < s["bias_len"].unsqueeze(1), at + 1, 0)
        last = zero.scatter_reduce(1, s["bias_ids"].long(), entry, "amax")
        bias = s["bias_values"].gather(1, (last - 1).clamp(min=0))
        x = torch.where(last > 0, x + bias, x)
    ok = None
    if s["allowed"] is not None:
        bits = (s["allowed"].unsqueeze(-1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        ok = bits.flatten(1)[:, :v] > 0
        x = torch.where(ok, x, float("-inf"))
    y = x.to(s["out"].dtype)
    best = y == y.amax(dim=1, keepdim=True)
    if ok is not None:
        best = best & ok
    i = torch.where(best, torch.arange(v, device="cuda"), v).amin(dim=1)  # the first of the largest
    return {"logits": y, "token": torch.where(i < v, i, -1).to(torch.int32)}


# ------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "logits":
        return {"logits": _exact_logits(s), "token": None}
    k, group = c["k"], c["group"]
    if c["op"] == "quantize":
        w = s["w"].double()
        values, scales = torch.empty_like(w), torch.empty(s["scales"].shape, dtype=torch.float64, device="cuda")
        for j in range(scales.shape[1]):
            part = w[:, j * group:(j + 1) * group]
            scale = (part.abs().max(dim=1).values / 7).to(torch.bfloat16).double()
            q = torch.round(part / scale.unsqueeze(1)).clamp(-8, 7)
            values[:, j * group:(j + 1) * group] = torch.nan_to_num(q) * scale.unsqueeze(1)
            scales[:, j] = scale
        return {"values": values, "scales": scales}
    if c["op"] == "embed":
        rows = s["rows"].long()
        return _exact_rows(s["codes"][rows], s["scales"][rows], k, group)
    x, parts = s["x"].double(), []
    for i in range(0, c["n"], 8192):
        parts.append(x @ _exact_rows(s["codes"][i:i + 8192], s["scales"][i:i + 8192], k, group).t())
    y = torch.cat(parts, dim=1)
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["residual"] is not None:
        y += s["residual"].double()
    return y


def _exact_rows(codes, scales, k, group):
    w = torch.empty((codes.shape[0], k), dtype=torch.float64, device="cuda")
    w[:, 0::2] = (codes % 16)[:, :(k + 1) // 2].double()
    w[:, 1::2] = (codes // 16)[:, :k // 2].double()
    w -= 8
    for j in range(scales.shape[1]):
        w[:, j * group:(j + 1) * group] *= scales[:, j:j + 1].double()
    return w


def _exact_logits(s):
    x = s["logits"].double()
    for i in range(x.shape[0]):
        row = x[i]
        n, p = int(s["history_len"][i]), int(s["prompt_len"][i])
        tokens = torch.unique(s["history"][i, :n].long())
        rep = s["repetition"][i].double()
        row[tokens] = torch.where(row[tokens] > 0, row[tokens] / rep, row[tokens] * rep)
        tokens, times = torch.unique(s["history"][i, p:n].long(), return_counts=True)
        row[tokens] -= s["frequency"][i].double() * times.double() + s["presence"][i].double()
        if s["bias_ids"] is not None:
            k = int(s["bias_len"][i])
            listed_ = dict(zip(s["bias_ids"][i, :k].tolist(), s["bias_values"][i, :k].tolist()))
            if listed_:
                row[torch.tensor(list(listed_), device="cuda")] += torch.tensor(
                    list(listed_.values()), dtype=torch.float64, device="cuda")
        if s["allowed"] is not None:
            word = s["allowed"][i].long()
            token = torch.arange(x.shape[1], device="cuda")
            row[(word[token // 32] >> (token % 32)) % 2 == 0] = float("-inf")
    return x
