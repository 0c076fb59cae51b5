"""Workloads of the 4-bit projections and of the cross attention, with their plain forms.

Three operators, used together in a conditioned transformer block that runs its
projections in 4 bits:

* ``quantize``: microscaled 4-bit quantisation of activations (and reading them back).
  A block of 32 (``mxfp4``: power-of-two scale) or 16 (``nvfp4``: e4m3 scale, times one
  scale of the tensor) consecutive columns shares a scale; values are e2m1.
* ``linear``: y = x W^T + b with W kept in 4 bits and x quantised on the way in.
* ``cross``: softmax attention of the tokens to an encoder's states of another length,
  heads grouped over fewer key/value heads, each sample with its own number of states.

``run`` computes the plain forms with elementary torch operations, or, with ``own``
set, calls the framework's operators.
"""
import math

import torch

own = False

HEAD_DIM = 128
BLOCK = {"mxfp4": 32, "nvfp4": 16}
WEIGHT_TENSOR_SCALE = 2.0 ** -8       # e4m3 block scales of weights ~N(0, 0.02) stay normal numbers


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _quantize(name, fmt, rows, cols):
    return {"name": name, "op": "quantize", "format": fmt, "rows": rows, "cols": cols}


def _linear(name, fmt, rows, cols, outs):
    return {"name": name, "op": "linear", "format": fmt, "rows": rows, "cols": cols, "outs": outs}


def _cross(name, batch, queries, states, heads, kv_heads, shared=False, ragged=False):
    return {"name": name, "op": "cross", "batch": batch, "queries": queries, "states": states, "heads": heads,
            "kv_heads": kv_heads, "shared": shared, "ragged": ragged}


def listed():
    return [
        # one conditioning row at model width: the smallest call, all latency
        _quantize("quantize_token", "mxfp4", 1, 5120),
        # the joint video + text sequence of a denoising step, before a block's projections
        _quantize("quantize_step", "nvfp4", 18944, 5120),
        # a ragged clip at an odd width: the last block of a row is partly filled
        _quantize("quantize_odd", "mxfp4", 777, 1795),
        # the QKV projection of one token: the weights are read for a single row
        _linear("linear_token", "nvfp4", 1, 5120, 15360),
        # an out-projection of the text tokens
        _linear("linear_text", "mxfp4", 512, 5120, 5120),
        # the gate-and-up projection of the whole sequence
        _linear("linear_step", "nvfp4", 18944, 5120, 27648),
        # sizes that end inside every tile
        _linear("linear_odd", "mxfp4", 333, 1795, 4861),
        # one new token of four samples, each with its own number of text states
        _cross("cross_token", 4, 1, 512, 40, 40, ragged=True),
        # one token of a sample over the tokens of a whole clip, grouped heads
        _cross("cross_token_long", 1, 1, 18432, 40, 8),
        # a clip's tokens over its text states: two samples of the same prompt
        _cross("cross_text", 2, 9216, 512, 40, 40, shared=True),
        # a padded batch of odd lengths with grouped heads; one sample has no states
        _cross("cross_ragged", 5, 1001, 777, 16, 4, ragged=True),
        # a clip's tokens over the tokens of a four-frame reference clip
        _cross("cross_clip", 1, 18432, 2304, 40, 40),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "cross"])
    fmt = rng.choice(["mxfp4", "nvfp4"])
    if op == "quantize":
        case = _quantize("", fmt, _log(rng, 1, 18944), _log(rng, 33, 5120))
    elif op == "linear":
        case = _linear("", fmt, _log(rng, 1, 18944), _log(rng, 100, 5120), _log(rng, 100, 27648))
    else:
        kv_heads = rng.choice([1, 2, 4, 8, 14, 40])
        heads = kv_heads * rng.choice([g for g in (1, 2, 4, 5, 7, 8) if g * kv_heads <= 40])
        batch = _log(rng, 1, 16)
        case = _cross("", batch, _log(rng, 1, max(1, 18432 // batch)), _log(rng, 1, 2304), heads, kv_heads,
                      shared=rng.random() < 0.25, ragged=rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(g, rows, cols):
    """Tokens after a norm: unit normal, with channels of different strength."""
    channel = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    return (torch.randn(rows, cols, generator=g, device="cuda") * channel).bfloat16()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "quantize":
        state["x"] = _activations(g, case["rows"], case["cols"])
    elif case["op"] == "linear":
        state["x"] = _activations(g, case["rows"], case["cols"])
        state["bias"] = torch.randn(case["outs"], generator=g, device="cuda").mul_(0.1).bfloat16()
        weight = (0.02 * torch.randn(case["outs"], case["cols"], generator=g, device="cuda")).bfloat16()
        # the weights as a 4-bit checkpoint holds them: two codes a byte, one scale byte a block
        fmt = case["format"]
        state["tensor_scale"] = WEIGHT_TENSOR_SCALE if fmt == "nvfp4" else 1.0
        index, sign, scale = _plain_codes(weight.float(), fmt, state["tensor_scale"])
        code = (index + 8 * sign).to(torch.uint8)
        code = torch.nn.functional.pad(code, (0, code.shape[1] % 2))
        state["codes"] = code[:, 0::2] | (code[:, 1::2] << 4)
        state["scales"] = ((torch.frexp(scale)[1] + 126).to(torch.uint8) if fmt == "mxfp4"
                           else scale.to(torch.float8_e4m3fn).view(torch.uint8))
        if own:
            import h3b200
            state["weight"] = h3b200.pack_fp4(state["codes"], state["scales"], fmt, cols=case["cols"],
                                              tensor_scale=state["tensor_scale"])
    else:
        batch, kv_batch = case["batch"], 1 if case["shared"] else case["batch"]
        state["q"] = torch.randn(batch, case["queries"], case["heads"], HEAD_DIM, generator=g, device="cuda").bfloat16()
        # the encoder's keys and values side by side, as one projection writes them
        kv = torch.randn(kv_batch, case["states"], 2, case["kv_heads"], HEAD_DIM, generator=g, device="cuda").bfloat16()
        state["k"], state["v"] = kv[:, :, 0], kv[:, :, 1]
        state["lengths"] = None
        if case["ragged"]:
            state["lengths"] = torch.randint(1, case["states"] + 1, (batch,), generator=g, device="cuda")
            state["lengths"][-1:] = 0 if batch > 1 else case["states"]
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _blocks(x, fmt):
    """x [rows, cols] in blocks of columns [rows, blocks, size], the last one filled with zeros."""
    size = BLOCK[fmt]
    return torch.nn.functional.pad(x, (0, -x.shape[1] % size)).view(x.shape[0], -1, size)


def _power(exponent):
    """2^exponent in fp32, from its bits (-127: the subnormal 2^-127)."""
    return torch.where(exponent < -126, 1 << 22, (exponent + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_codes(x, fmt, tensor_scale):
    """Magnitude code (0..7), sign and block scale of x (fp32). A power of two divides exactly,
    and x / scale of an 8-bit and a 4-bit significand is never rounded onto a border it is not on."""
    b = _blocks(x, fmt)
    amax = b.abs().amax(-1)
    if fmt == "mxfp4":
        # 2^(floor(log2 amax) - 2): e2m1's largest value is 1.5 * 2^2
        scale = _power(((amax.view(torch.int32) >> 23) - 129).clamp(-127, 127))
        ratio = b / scale[..., None]
    else:
        scale = (amax / torch.full_like(amax, 6 * tensor_scale)).clamp(max=448).to(torch.float8_e4m3fn).float()
        ratio = torch.where(scale[..., None] > 0, b / (scale * tensor_scale)[..., None], 0)
    a = ratio.abs()
    # borders between 0, .5, 1, 1.5, 2, 3, 4, 6; a tie goes to the even code
    index = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)).flatten(1)
    sign = (ratio < 0).int().flatten(1)
    return index[:, : x.shape[1]], sign[:, : x.shape[1]], scale


def _plain_values(index, sign, scale, fmt, tensor_scale):
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=index.device)[index] * (1 - 2 * sign)
    return (_blocks(value, fmt) * (scale * tensor_scale)[..., None]).flatten(1)[:, : index.shape[1]]


def _plain_weight(state):
    byte, fmt = state["codes"].int(), state["format"]
    code = torch.stack((byte & 15, byte >> 4), -1).flatten(1)[:, : state["cols"]]
    scale = (_power(state["scales"].int() - 127) if fmt == "mxfp4"
             else state["scales"].view(torch.float8_e4m3fn).float())
    return _plain_values(code & 7, code >> 3, scale, fmt, state["tensor_scale"])


def _plain_cross(q, k, v, lengths):
    batch, queries, heads, dim = q.shape
    kv_heads, states = k.shape[2], k.shape[1]
    k = k.float().expand(batch, -1, -1, -1).permute(0, 2, 3, 1)[:, :, None]        # [B, Hkv, 1, D, Sk]
    v = v.float().expand(batch, -1, -1, -1).permute(0, 2, 1, 3)[:, :, None]        # [B, Hkv, 1, Sk, D]
    q = q.float().view(batch, queries, kv_heads, -1, dim).permute(0, 2, 3, 1, 4)   # [B, Hkv, G, Sq, D]
    score = torch.matmul(q, k).mul_(dim ** -0.5)
    if lengths is not None:
        past = torch.arange(states, device=q.device) >= lengths[:, None]
        score.masked_fill_(past[:, None, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)   # a row without states has none
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / torch.where(total > 0, total, 1)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, dim).bfloat16()


def run(state):
    op = state["op"]
    if own:
        import h3b200
        if op == "quantize":
            return h3b200.dequantize_fp4(h3b200.quantize_fp4(state["x"], state["format"]))
        if op == "linear":
            return h3b200.linear_fp4(state["x"], state["weight"], bias=state["bias"])
        return h3b200.cross_attention(state["q"], state["k"], state["v"], lengths=state["lengths"])
    if op == "cross":
        return _plain_cross(state["q"], state["k"], state["v"], state["lengths"])
    fmt = state["format"]
    x = _plain_values(*_plain_codes(state["x"].float(), fmt, 1.0), fmt, 1.0)
    if op == "quantize":
        return x.bfloat16()
    return (torch.matmul(x, _plain_weight(state).t()) + state["bias"].float()).bfloat16()


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_power(exponent):
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_quantize(x, fmt):
    rows, cols = x.shape
    size = BLOCK[fmt]
    padded = torch.zeros(rows, -(-cols // size) * size, dtype=torch.float64, device=x.device)
    padded[:, :cols] = x.double()
    group = padded.unflatten(1, (-1, size))
    largest = group.abs().max(-1, keepdim=True).values
    if fmt == "mxfp4":
        # floor(log2 a) = frexp's exponent - 1; a block of zeros takes the smallest scale
        exponent = torch.where(largest > 0, torch.frexp(largest)[1] - 3, -127).clamp(-127, 127)
        scale = _exact_power(exponent)
    else:
        # e4m3: 3 bits behind the leading one, exponents from -6, ties to even, at most 448
        sixth = largest / torch.full_like(largest, 6)
        step = _exact_power((torch.frexp(sixth)[1] - 1).clamp(min=-6) - 3)
        scale = (torch.round(sixth / step) * step).clamp(max=448)
    ratio = torch.where(scale > 0, group / scale, torch.zeros_like(group))
    size_of = ratio.abs().clamp(max=6)
    # e2m1's values lie 1/2 apart below 2, 1 apart below 4, 2 apart up to 6; round() takes ties to even
    apart = torch.where(size_of < 2, 0.5, torch.where(size_of < 4, 1.0, 2.0)).double()
    value = torch.round(size_of / apart) * apart * torch.sign(ratio) * scale
    return value.flatten(1)[:, :cols]


def _exact_weight(state):
    low, high = state["codes"] % 16, torch.div(state["codes"], 16, rounding_mode="floor")
    code = torch.empty(low.shape[0], 2 * low.shape[1], dtype=torch.float64, device=low.device)
    code[:, 0::2], code[:, 1::2] = low.double(), high.double()
    code = code[:, : state["cols"]]
    magnitude = code % 8
    exponent, half = torch.div(magnitude, 2, rounding_mode="floor"), (magnitude % 2) / 2
    value = torch.where(exponent == 0, half, (1 + half) * _exact_power(exponent - 1))
    value = torch.where(code >= 8, -value, value)
    byte = state["scales"].double()
    if state["format"] == "mxfp4":
        scale = _exact_power(byte - 127)
    else:
        exponent, part = torch.div(byte, 8, rounding_mode="floor"), (byte % 8) / 8
        scale = torch.where(exponent == 0, part * 2.0 ** -6, (1 + part) * _exact_power(exponent - 7))
        scale = scale * state["tensor_scale"]
    return value * scale.repeat_interleave(BLOCK[state["format"]], 1)[:, : state["cols"]]


def _exact_cross(state):
    q, k, v = (state[n].double() for n in "qkv")
    group = q.shape[2] // k.shape[2]
    out = torch.zeros_like(q)
    for b in range(q.shape[0]):
        kb, vb = (t[b if t.shape[0] > 1 else 0] for t in (k, v))
        n = kb.shape[0] if state["lengths"] is None else int(state["lengths"][b])
        if n == 0:
            continue
        for h in range(q.shape[2]):
            score = q[b, :, h] @ kb[:n, h // group].t() / math.sqrt(q.shape[3])
            out[b, :, h] = torch.softmax(score, -1) @ vb[:n, h // group]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "cross":
        return _exact_cross(state)
    x = _exact_quantize(state["x"], case["format"])
    if case["op"] == "quantize":
        return x
    return x @ _exact_weight(state).t() + state["bias"].double()


def work(case):
    if case["op"] == "cross":
        q = case["batch"] * case["queries"] * case["heads"] * HEAD_DIM
        kv = (1 if case["shared"] else case["batch"]) * case["states"] * case["kv_heads"] * HEAD_DIM
        return {"bytes": 2 * (2 * q + 2 * kv), "flops": 4 * q * case["states"]}
    rows, cols = case["rows"], case["cols"]
    held = rows * cols / 2 + rows * -(-cols // BLOCK[case["format"]])       # codes and scales
    if case["op"] == "quantize":
        # x read, codes and scales written and read back, the values written
        return {"bytes": 4 * rows * cols + 2 * held, "flops": 4 * rows * cols}
    outs = case["outs"]
    weight = outs * cols / 2 + outs * -(-cols // BLOCK[case["format"]])
    return {"bytes": 2 * rows * cols + weight + 2 * outs + 2 * rows * outs, "flops": 2 * rows * cols * outs}
