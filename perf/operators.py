"""What the transformer-block operators are measured on: RMSNorm with the residual's addition and a
quantised output, microscaled 4-bit (MXFP4) quantisation and product, and attention with a sliding
window and first tokens that stay visible.

`run` computes one call of an operator, in plain torch operations or, with `own` set, by the calls a
user of the package makes.  Formulas (bf16 in and out, everything between in 32 bits):

  norm       r = bf16(x + residual);  y = r / sqrt(mean(r^2) + eps) * weight, then quantised:
             int8   scale = max|y| / 127 per row (at least 1e-30), q = round half even(y / scale)
             mxfp4  as below, per 32 columns
  mxfp4      per 32 consecutive columns: e = floor(log2(max|x|)) - 2 within [-127, 127] (-127 where
             all are zero), stored as the byte e + 127; element = x / 2^e rounded to the nearest of
             +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ties to the even code, saturating; two per byte, the
             even column in the low half.  Scale bytes lie in tiles of 128 rows x 4 blocks:
             [row tile][column tile][row % 32][row % 128 // 32][block % 4]
  product    out = bf16(a @ w.T + bias) of two such matrices
  attention  query i of a batch entry with n keys sits at p = i + n - q_len; it sees the keys j < n
             with j <= p + right and (j >= p - left or j < sinks); left or right -1: no limit on
             that side; a query that sees no key gives zeros
"""
import importlib

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
HEAD_DIM = 128
#: the values of the 16 codes of a 4-bit element
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def ops():
    return importlib.import_module("dcu-video-dit-turbo_b200").ops


def listed():
    return [
        # one token of a serving loop enters a layer: latency counts
        dict(name="norm_int8_one_token", kind="norm", rows=1, columns=3072, form="int8", residual=True),
        # the block's whole token stream of a 28-frame clip at 22 x 38 latent positions
        dict(name="norm_int8_clip", kind="norm", rows=23638, columns=3072, form="int8", residual=True),
        # a wider layer, an odd number of tokens, straight into the 4-bit product's format
        dict(name="norm_mxfp4_odd", kind="norm", rows=4099, columns=5120, form="mxfp4", residual=True),
        # attention rows on their way into the output projection
        dict(name="quantize_clip", kind="quantize", rows=23638, columns=3072, act="none"),
        # the feed-forward's second projection: SwiGLU and quantisation of one rank's tokens
        dict(name="quantize_swiglu", kind="quantize", rows=5910, columns=8192, act="swiglu"),
        # a few conditioning tokens through the packed projection: the weights are all the traffic
        dict(name="product_few_rows", kind="product", rows=8, outputs=9216, columns=3072, bias=True, quantized=True),
        # ragged everywhere: a shard's tail, an output width and a depth that fill no tile
        dict(name="product_ragged", kind="product", rows=1537, outputs=1000, columns=2080, bias=False, quantized=True),
        # the packed projection of a whole clip, from bf16 activations
        dict(name="linear_clip", kind="product", rows=23638, outputs=9216, columns=3072, bias=True, quantized=False),
        # a clip that attends to four frames on each side and to its first frame throughout
        dict(name="attention_clip", kind="attention", batch=1, heads=24, kv_heads=24, q_len=23638, kv_len=23638,
             left=3344, right=3344, sinks=836, ragged=False),
        # causal, shared key heads, two padded sequences of odd length
        dict(name="attention_causal_shared_heads", kind="attention", batch=2, heads=24, kv_heads=8, q_len=4099,
             kv_len=4099, left=1023, right=0, sinks=4, ragged=True),
        # the next frame's tokens against a long cache
        dict(name="attention_next_frame", kind="attention", batch=1, heads=24, kv_heads=24, q_len=836, kv_len=24244,
             left=8360, right=836, sinks=836, ragged=False),
        # single tokens of a batch of sequences of different lengths
        dict(name="attention_single_tokens", kind="attention", batch=8, heads=24, kv_heads=6, q_len=1, kv_len=16411,
             left=4095, right=0, sinks=128, ragged=True),
    ]


def _log(rng, low, high):
    """A whole number between low and high, evenly over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("norm", "quantize", "product", "attention", "attention"))
    if kind == "norm":
        form = rng.choice(("int8", "mxfp4"))
        rows = _log(rng, 1, 23638)
        columns = _log(rng, 32, 8192)
        columns = columns // 32 * 32 if form == "mxfp4" else columns if rng.random() < 0.2 else max(8, columns // 8 * 8)
        return dict(kind=kind, rows=min(rows, 60_000_000 // columns), columns=columns, form=form, residual=rng.random() < 0.8)
    if kind == "quantize":
        columns = _log(rng, 1, 256) * 32
        return dict(kind=kind, rows=min(_log(rng, 1, 23638), 40_000_000 // columns), columns=columns,
                    act=rng.choice(("none", "swiglu")))
    if kind == "product":
        return dict(kind=kind, rows=_log(rng, 1, 16384), outputs=_log(rng, 1, 1152) * 8, columns=_log(rng, 1, 128) * 32,
                    bias=rng.random() < 0.5, quantized=rng.random() < 0.5)
    kv_heads = rng.choice((1, 2, 3, 6, 8, 12, 24))
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if kv_heads * g <= 24])
    batch = rng.choice((1, 1, 2, 3, 8))
    kv_len = _log(rng, 1, 16384)
    form = rng.choice(("one", "few", "chunk", "all"))
    q_len = {"one": 1, "few": rng.randint(2, 16), "chunk": _log(rng, 16, 2048), "all": kv_len}[form]
    q_len = max(1, min(q_len, 2_000_000_000 // (batch * heads * kv_len)))
    left = rng.choice((-1, 0, _log(rng, 1, 8192), _log(rng, 64, 4096)))
    right = rng.choice((0, 0, -1, _log(rng, 1, 4096)))
    return dict(kind="attention", batch=batch, heads=heads, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len, left=left,
                right=right, sinks=rng.choice((0, 1, 4, _log(rng, 8, 1024))), ragged=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs

def _activations(rows, columns, g):
    """Normal values with a few channels that are an order of magnitude larger, as hidden states have."""
    x = torch.randn((rows, columns), generator=g, device=DEVICE)
    loud = torch.randint(0, columns, (max(1, columns // 256),), generator=g, device=DEVICE)
    x[:, loud] *= 12.0
    return x.bfloat16()


def _random_mxfp4(rows, columns, g):
    """A quantised matrix as a program holds it: packed elements, scale bytes in tiles (padding is zero)."""
    q = torch.randint(0, 256, (rows, columns // 2), generator=g, device=DEVICE, dtype=torch.uint8)
    e = torch.randint(118, 125, (rows, columns // 32), generator=g, device=DEVICE, dtype=torch.uint8)
    row_tiles, column_tiles = -(-rows // 128), -(-columns // 128)
    full = torch.zeros((row_tiles * 128, column_tiles * 4), device=DEVICE, dtype=torch.uint8)
    full[:rows, :columns // 32] = e
    s = full.view(row_tiles, 4, 32, column_tiles, 4).permute(0, 3, 2, 1, 4).reshape(row_tiles, column_tiles, 512).contiguous()
    return q, s


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, state = case["kind"], dict(case)
    if kind == "norm":
        state["x"] = _activations(case["rows"], case["columns"], g)
        state["r"] = _activations(case["rows"], case["columns"], g) if case["residual"] else None
        state["w"] = (1.0 + 0.1 * torch.randn((case["columns"],), generator=g, device=DEVICE)).bfloat16()
    elif kind == "quantize":
        state["x"] = _activations(case["rows"], case["columns"] * (2 if case["act"] == "swiglu" else 1), g)
    elif kind == "product":
        if case["quantized"]:
            state["a"], state["a_scale"] = _random_mxfp4(case["rows"], case["columns"], g)
        else:
            state["x"] = _activations(case["rows"], case["columns"], g)
        state["w"], state["w_scale"] = _random_mxfp4(case["outputs"], case["columns"], g)
        state["b"] = torch.randn((case["outputs"],), generator=g, device=DEVICE).bfloat16() if case["bias"] else None
    else:
        batch, heads, kv_heads, q_len, kv_len = (case[k] for k in ("batch", "heads", "kv_heads", "q_len", "kv_len"))
        normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE).bfloat16()  # noqa: E731
        if batch == 1 and heads == kv_heads and q_len == kv_len:   # a packed projection's output
            packed = normal(q_len, 3, heads, HEAD_DIM)
            state["q"], state["k"], state["v"] = (packed[:, i].transpose(0, 1).unsqueeze(0) for i in range(3))
        else:                                                      # a cache of [batch, kv_len, head] rows
            state["q"] = normal(batch, q_len, heads, HEAD_DIM).transpose(1, 2)
            state["k"] = normal(batch, kv_len, kv_heads, HEAD_DIM).transpose(1, 2)
            state["v"] = normal(batch, kv_len, kv_heads, HEAD_DIM).transpose(1, 2)
        state["lengths"] = None
        if case["ragged"]:
            lengths = torch.randint(kv_len // 2, kv_len + 1, (batch,), generator=g, device=DEVICE, dtype=torch.int32)
            lengths[0] = kv_len
            state["lengths"] = lengths
    return state


# ---------------------------------------------------------------- the plain forms

def _values_of(q, s, rows, columns):
    """The fp32 values of a quantised matrix."""
    table = torch.tensor(CODES, device=q.device)
    elements = torch.stack((table[(q & 15).long()], table[(q >> 4).long()]), dim=-1).view(rows, columns // 32, 32)
    e = s.view(s.shape[0], s.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, s.shape[1] * 4)
    e = e[:rows, :columns // 32].int() - 127
    return torch.ldexp(elements, e.unsqueeze(-1)).view(rows, columns)


def _round_mxfp4(x):
    """The values that an fp32 matrix has after quantisation."""
    blocks = x.view(x.shape[0], -1, 32)
    largest = blocks.abs().amax(-1, keepdim=True)
    e = torch.where(largest > 0, torch.frexp(largest)[1] - 3, -127).clamp(-127, 127)
    a = torch.ldexp(blocks, -e)
    size = a.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    rounded = ((size / step).round() * step).clamp(max=6.0)
    return torch.ldexp(torch.copysign(rounded, a), e).view(x.shape)


def _plain_norm(state):
    x = state["x"].float()
    if state["r"] is not None:
        x = (x + state["r"].float()).bfloat16().float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * state["w"].float()
    if state["form"] == "mxfp4":
        values = _round_mxfp4(y)
    else:
        scale = (y.abs().amax(-1, keepdim=True) / 127.0).clamp(min=1e-30)
        values = (y / scale).round().clamp(-127, 127) * scale
    return dict(values=values.bfloat16(), summed=x.bfloat16())


def _plain_quantize(state):
    x = state["x"].float()
    if state["act"] == "swiglu":
        gate, up = x.chunk(2, dim=-1)
        x = gate / (1.0 + torch.exp(-gate)) * up
    return _round_mxfp4(x.contiguous()).bfloat16()


def _plain_product(state):
    rows, outputs, columns = state["rows"], state["outputs"], state["columns"]
    a = _values_of(state["a"], state["a_scale"], rows, columns) if state["quantized"] else _round_mxfp4(state["x"].float())
    out = a @ _values_of(state["w"], state["w_scale"], outputs, columns).t()
    if state["b"] is not None:
        out += state["b"].float()
    return out.bfloat16()


def _plain_attention(state):
    q, k, v = state["q"].float(), state["k"].float(), state["v"].float()
    batch, heads, q_len, d = q.shape
    kv_heads, kv_len = k.shape[1], k.shape[2]
    n = state["lengths"] if state["lengths"] is not None else torch.full((batch,), kv_len, device=q.device)
    p = torch.arange(q_len, device=q.device)[None, :, None] + (n[:, None, None] - q_len)
    j = torch.arange(kv_len, device=q.device)[None, None, :]
    hidden = j >= n[:, None, None]
    if state["right"] >= 0:
        hidden = hidden | (j > p + state["right"])
    if state["left"] >= 0:
        hidden = hidden | ((j < p - state["left"]) & (j >= state["sinks"]))
    s = q.reshape(batch, kv_heads, -1, d) @ k.transpose(-1, -2)
    s = s.view(batch, heads, q_len, kv_len).mul_(d ** -0.5).masked_fill_(hidden.expand(batch, q_len, kv_len)[:, None], float("-inf"))
    largest = s.amax(-1, keepdim=True)
    s.sub_(torch.where(largest == float("-inf"), 0.0, largest)).exp_()
    total = s.sum(-1, keepdim=True)
    out = (s.view(batch, kv_heads, -1, kv_len) @ v).view(batch, heads, q_len, d)
    return (out / torch.where(total == 0, 1.0, total)).bfloat16()


def run(state):
    kind = state["kind"]
    if not own:
        return dict(norm=_plain_norm, quantize=_plain_quantize, product=_plain_product, attention=_plain_attention)[kind](state)
    o = ops()
    if kind == "norm":
        if state["form"] == "mxfp4":
            q, s, summed = o.rmsnorm_residual_mxfp4(state["x"], state["r"], state["w"], EPS)
            return dict(values=o.dequantize_mxfp4(q, s), summed=summed)
        q, s, summed = o.rmsnorm_residual_quant(state["x"], state["r"], state["w"], EPS)
        return dict(values=o.dequantize_int8_rowwise(q, s), summed=summed)
    if kind == "quantize":
        q, s = (o.swiglu_quantize_mxfp4 if state["act"] == "swiglu" else o.quantize_mxfp4)(state["x"])
        return o.dequantize_mxfp4(q, s)
    if kind == "product":
        if state["quantized"]:
            return o.mxfp4_gemm(state["a"], state["a_scale"], state["w"], state["w_scale"], state["b"])
        return o.mxfp4_linear(state["x"], state["w"], state["w_scale"], state["b"])
    return o.window_fwd_bhsd(state["q"], state["k"], state["v"], HEAD_DIM ** -0.5, state["left"], state["right"],
                             state["sinks"], state["lengths"])


# ---------------------------------------------------------------- what a pass cannot do without

def _visible_pairs(case, n):
    """How many (query, key) pairs of a sequence of n keys are visible, without a loop over the keys."""
    p = torch.arange(case["q_len"], dtype=torch.int64) + (n - case["q_len"])
    last = torch.full_like(p, n - 1) if case["right"] < 0 else (p + case["right"]).clamp(max=n - 1)
    first = torch.zeros_like(p) if case["left"] < 0 else (p - case["left"]).clamp(min=0)
    window = (last - first + 1).clamp(min=0)
    sinks = (torch.minimum(torch.minimum(first, last + 1), torch.full_like(p, min(case["sinks"], n)))).clamp(min=0)
    return int((window + sinks).sum()), int(torch.minimum(window + sinks, torch.tensor(n)).amax())


def work(case):
    kind = case["kind"]
    if kind == "norm":
        m, c = case["rows"], case["columns"]
        # x, residual and weight in; the sum (where there is one) and the quantised form's values out
        return dict(bytes=2 * m * c * (4 if case["residual"] else 2) + 2 * c, flops=6 * m * c)
    if kind == "quantize":
        m, k = case["rows"], case["columns"]
        return dict(bytes=2 * m * k * (3 if case["act"] == "swiglu" else 2), flops=4 * m * k)
    if kind == "product":
        m, n, k = case["rows"], case["outputs"], case["columns"]
        packed = k // 2 + k // 32
        return dict(bytes=(m * packed if case["quantized"] else 2 * m * k) + n * packed + 2 * m * n + (2 * n if case["bias"] else 0),
                    flops=2 * m * n * k)
    b, h, hk, sq = case["batch"], case["heads"], case["kv_heads"], case["q_len"]
    # ragged lengths lie evenly between half and all of the keys
    lengths = [case["kv_len"]] + [case["kv_len"] * 3 // 4 if case["ragged"] else case["kv_len"]] * (b - 1)
    pairs, keys = 0, 0
    for n in lengths:
        found, most = _visible_pairs(case, n)
        pairs += found
        keys += min(n, most + sq - 1)
    return dict(bytes=2 * HEAD_DIM * (2 * b * h * sq + 2 * hk * keys), flops=4 * HEAD_DIM * h * pairs)


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_mxfp4(y):
    """Values after 4-bit quantisation, by the distance to every code."""
    shape, y = y.shape, y.reshape(-1, 32)
    out = torch.empty_like(y)
    sizes = torch.tensor(CODES[:8], dtype=torch.float64, device=y.device)
    borders = (sizes[1:] + sizes[:-1]) / 2
    for at in range(0, y.shape[0], 1 << 20):
        part = y[at:at + (1 << 20)]
        largest = part.abs().amax(1)
        e = torch.floor(torch.log2(torch.where(largest > 0, largest, 1.0)))
        e = torch.where(torch.exp2(e) > largest, e - 1, torch.where(torch.exp2(e + 1) <= largest, e + 1, e)) - 2
        unit = torch.exp2(torch.where(largest > 0, e, -127.0).clamp(-127, 127))[:, None]
        a = part.abs() / unit
        below = torch.bucketize(a, borders)                  # the borders < a
        tie = (below < 7) & (a == borders[below.clamp(max=6)])
        code = torch.where(tie & (below % 2 == 1), below + 1, below)
        out[at:at + (1 << 20)] = torch.sign(part) * sizes[code] * unit
    return out.view(shape)


def _exact_packed(q, s, rows, columns):
    at = torch.arange(rows, device=q.device)[:, None]
    block = torch.arange(columns // 32, device=q.device)[None, :]
    byte = s[at // 128, block // 4, at % 32 * 16 + at % 128 // 32 * 4 + block % 4]
    values = torch.empty((rows, columns), dtype=torch.float64, device=q.device)
    table = torch.tensor(CODES, dtype=torch.float64, device=q.device)
    values[:, 0::2] = table[(q % 16).long()]
    values[:, 1::2] = table[(q // 16).long()]
    return values * torch.exp2(byte.double() - 127).repeat_interleave(32, dim=1)


def _exact_attention(state, case):
    q, k, v = state["q"], state["k"], state["v"]
    batch, heads, q_len, d = q.shape
    kv_len, share = k.shape[2], heads // k.shape[1]
    out = torch.zeros((batch, heads, q_len, d), dtype=torch.float64, device=q.device)
    for b in range(batch):
        n = kv_len if state["lengths"] is None else int(state["lengths"][b])
        if n == 0:
            continue
        keys = torch.arange(n, device=q.device)
        for i0 in range(0, q_len, 8192):
            i1 = min(q_len, i0 + 8192)
            p = torch.arange(i0, i1, device=q.device)[:, None] + n - q_len
            seen = torch.ones((i1 - i0, n), dtype=torch.bool, device=q.device)
            if case["left"] >= 0:
                seen &= (keys >= p - case["left"]) | (keys < case["sinks"])
            if case["right"] >= 0:
                seen &= keys <= p + case["right"]
            some = seen.any(1)
            for h in range(heads):
                score = q[b, h, i0:i1].double() @ k[b, h // share, :n].double().t() / d ** 0.5
                score[~seen] = float("-inf")
                score[~some] = 0.0
                weight = torch.softmax(score, dim=1)
                out[b, h, i0:i1] = (weight @ v[b, h // share, :n].double()) * some[:, None]
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "attention" and case["batch"] * case["heads"] * case["q_len"] * case["kv_len"] > 16_000_000_000:
        return None
    state = prepare(case, seed)
    if kind == "norm":
        x = state["x"].double()
        if state["r"] is not None:
            x = (x + state["r"].double()).bfloat16().double()
        y = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * state["w"].double()
        if case["form"] == "mxfp4":
            return dict(values=_exact_mxfp4(y), summed=x)
        unit = (y.abs().amax(1, keepdim=True) / 127).clamp(min=1e-30)
        return dict(values=torch.round(y / unit) * unit, summed=x)
    if kind == "quantize":
        x = state["x"].double()
        if case["act"] == "swiglu":
            gate, up = x[:, :case["columns"]], x[:, case["columns"]:]
            x = gate * torch.sigmoid(gate) * up
        return _exact_mxfp4(x.contiguous())
    if kind == "product":
        if case["quantized"]:
            a = _exact_packed(state["a"], state["a_scale"], case["rows"], case["columns"])
        else:
            a = _exact_mxfp4(state["x"].double())
        out = a @ _exact_packed(state["w"], state["w_scale"], case["outputs"], case["columns"]).t()
        return out if state["b"] is None else out + state["b"].double()
    return _exact_attention(state, case)
