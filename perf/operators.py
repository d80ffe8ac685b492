"""The operators of the 8-bit transformer path, as measured: each case's inputs, the call a user makes and its plain form.

* ``linear``: a matrix product in 8-bit integers with a scale per token and per channel (``int8_linear``).  The tokens
  come in 16 bits and are quantised in the call, or (``rows = "int8"``) are already codes and scales; ``joined`` > 0
  splits the inner axis over two sources, as the single-stream output projection takes [attention | MLP].
* ``modulated``: the adaptive LayerNorm in front of a projection, with the tokens quantised in the same pass
  (``adaln_int8``; with the gated residual ``gate_residual_adaln_int8``), then the product.
* ``qk``: RMSNorm of query and key heads with the rotary embedding, both in one pass (``norm_rope_qk``).

Quantisation of a row: scale = max|x| / 127, code = round(x * (127 / max|x|)), ties to even.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    linear = dict(op="linear", dtype="bf16", bias=True, act=False, rows="16bit", joined=0)
    mod = dict(op="modulated", dtype="bf16", batch=1, residual=True, act=False)
    qk = dict(op="qk", dtype="bf16", batch=1, text=0)
    return [
        # the pooled-text embedder of two prompts: the smallest call of a step, latency alone
        dict(linear, name="embedder 2 tokens", m=2, k=768, n=3072, dtype="fp16"),
        # a double-stream block's modulation from the conditioning vector: one token, the weights are all there is to read
        dict(linear, name="modulation 1 token", m=1, k=3072, n=18432),
        # Q, K and V of the 512 text tokens, joined in one product
        dict(linear, name="text qkv 512", m=512, k=3072, n=9216),
        # nothing even: odd tokens, channels and inner size
        dict(linear, name="odd 1771x1333x1001", m=1771, k=1001, n=1333, dtype="fp16", act=True),
        # the image stream's MLP input at 2048 x 2048 pixels
        dict(linear, name="mlp in 16384", m=16384, k=3072, n=12288, act=True),
        # Q, K and V of the joined stream from tokens that are codes already (the modulation quantised them)
        dict(linear, name="qkv 16896 codes", m=16896, k=3072, n=9216, rows="int8"),
        # the single-stream output projection over [attention | MLP]: the longest inner axis
        dict(linear, name="joined out 16896", m=16896, k=15360, n=3072, joined=3072),
        # a small block of two images, ragged tokens, no residual
        dict(mod, name="modulated 2x77", batch=2, tokens=77, c=256, n=1000, dtype="fp16", residual=False),
        # residual, modulation and MLP input of the image stream at 1024 x 1024 pixels
        dict(mod, name="modulated 4096", tokens=4096, c=3072, n=12288, act=True),
        # one token's queries and keys
        dict(qk, name="qk 1 token", tokens=1, hq=24, hk=24, d=128),
        # shared key heads, 64 wide, three ragged sequences
        dict(qk, name="qk 3x1013 shared", batch=3, tokens=1013, hq=20, hk=4, d=64, dtype="fp16"),
        # queries and keys of the joined stream at 2048 x 2048 pixels, text rows with their own weights
        dict(qk, name="qk 16896", tokens=16896, hq=24, hk=24, d=128, text=512),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "modulated", "qk"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "linear":
        while True:
            m, k, n = _spread(rng, 1, 20000), _spread(rng, 64, 16000), _spread(rng, 16, 24000)
            if m * k * n <= 16896 * 15360 * 3072 and n * k <= 1 << 28 and m * n <= 1 << 28:
                break
        if rng.random() < 0.6:  # widths of models are seldom odd
            k, n = max(64, k // 64 * 64), max(16, n // 16 * 16)
        rows = rng.choice(["16bit", "16bit", "int8"])
        joined = rng.randrange(8, k - 8) // 8 * 8 if rows == "16bit" and rng.random() < 0.25 else 0
        return dict(op=op, dtype=dtype, bias=rng.random() < 0.7, act=rng.random() < 0.3, rows=rows, joined=joined,
                    m=m, k=k, n=n)
    if op == "modulated":
        while True:
            batch, tokens, c, n = rng.randint(1, 4), _spread(rng, 1, 17000), 256 * rng.randint(1, 16), _spread(rng, 16, 24000)
            if batch * tokens * c * n <= 16896 * 15360 * 3072 and batch * tokens * n <= 1 << 28:
                break
        return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, c=c, n=n, residual=rng.random() < 0.6,
                    act=rng.random() < 0.4)
    while True:
        batch, tokens, d = rng.randint(1, 4), _spread(rng, 1, 20000), rng.choice([64, 128, 256])
        hk = rng.randint(1, 24)
        hq = hk * rng.choice([1, 1, 2, 4])
        if batch * tokens * (hq + hk) * d <= 16896 * 48 * 128:
            break
    return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, hq=hq, hk=hk, d=d, text=rng.choice([0, tokens // 3]))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, width):
    """Tokens as a transformer block sees them: channels of unlike size, a few of them large."""
    channel = torch.exp(0.5 * _normal(g, width))
    return _normal(g, rows, width) * channel


def _padded(rows, width, dtype):
    """[rows, width] whose rows start on 16-byte boundaries."""
    step = 16 // torch.empty(0, dtype=dtype).element_size()
    return torch.zeros(rows, -(-width // step) * step, dtype=dtype, device="cuda")[:, :width]


def _codes(x):
    top = x.abs().amax(-1, keepdim=True)
    codes = _padded(x.shape[0], x.shape[1], torch.int8)
    codes.copy_(torch.round(x * (127.0 / top)))
    return codes, (top / 127.0)[:, 0].contiguous()


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "qk":
        b, t, hq, hk, d = (case[x] for x in ("batch", "tokens", "hq", "hk", "d"))
        joint = (2.0 * _normal(g, b, t, (hq + 2 * hk) * d)).to(dt)  # the joined projection's output
        s["q"] = joint[..., :hq * d].unflatten(-1, (hq, d))
        s["k"] = joint[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
        names = ("weight_q", "weight_k") + (("weight_txt_q", "weight_txt_k") if case["text"] else ())
        s["weights"] = {w: (1 + 0.1 * _normal(g, d)).to(dt) for w in names}
        half = torch.rand(t, d // 2, generator=g, device="cuda", dtype=torch.float64) * 128 * math.pi
        s["cos"], s["sin"] = (f(half).repeat_interleave(2, dim=1).float() for f in (torch.cos, torch.sin))
        return s
    if case["op"] == "modulated":
        b, t, k = case["batch"], case["tokens"], case["c"]
        s["x"] = (_activations(g, b * t, k) + 0.3).view(b, t, k).to(dt)
        s["shift"], s["scale"], s["gate"] = (0.5 * _normal(g, b, 3 * k)).to(dt).chunk(3, dim=-1)
        if case["residual"]:
            s["y"] = _activations(g, b * t, k).view(b, t, k).to(dt)
    else:
        m, k, j = case["m"], case["k"], case["joined"]
        if case["rows"] == "int8":
            s["codes"], s["code_scales"] = _codes(_activations(g, m, k).to(dt).float())
        elif j:
            s["a"], s["b"] = _activations(g, m, j).to(dt), _activations(g, m, k - j).to(dt)
        else:
            s["x"] = _activations(g, m, k).to(dt)
    s["w"], s["w_scales"] = _codes(_normal(g, case["n"], k))
    s["w_scales"] *= 1 / math.sqrt(k)
    s["bias_"] = (0.1 * _normal(g, case["n"])).to(dt) if case.get("bias", True) else None
    return s


def _own(s):
    import hilberta_b200 as hb
    from hilberta_b200 import block_ops

    dt = DTYPES[s["dtype"]]
    if s["op"] == "qk":
        return hb.norm_rope_qk(s["q"], s["k"], cos=s["cos"], sin=s["sin"], text_tokens=s["text"], **s["weights"])
    weight = hb.Int8Rows(s["w"], s["w_scales"], dt)
    kw = dict(bias=s["bias_"], activation="gelu_tanh" if s["act"] else None)
    if s["op"] == "modulated":
        if s["residual"]:
            x, rows = block_ops.gate_residual_adaln_int8(s["x"], s["y"], s["gate"], s["shift"], s["scale"],
                                                         x_out=torch.empty_like(s["x"]))
            return x, hb.int8_linear(rows, weight, **kw)
        return hb.int8_linear(block_ops.adaln_int8(s["x"], s["shift"], s["scale"]), weight, **kw)
    if s["rows"] == "int8":
        return hb.int8_linear(hb.Int8Rows(s["codes"], s["code_scales"], dt), weight, **kw)
    if s["joined"]:
        return hb.int8_linear(hb.quantize_rows(s["a"], joined=s["b"]), weight, **kw)
    return hb.int8_linear(s["x"], weight, **kw)


def _quantised(x):
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127.0 / top)), top / 127.0


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _product(s, codes, scales):
    out = codes @ s["w"].float().t() * (scales * s["w_scales"])
    if s["bias_"] is not None:
        out = out + s["bias_"].float()
    return (_gelu(out) if s["act"] else out).to(DTYPES[s["dtype"]])


def _rotated(x, weight, txt_weight, s):
    """RMSNorm over the last axis, then pairs (2i, 2i + 1) turned, in 32 bits."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    w = weight.float().expand(x.shape[1], 1, -1)
    if txt_weight is not None:
        w = torch.cat([txt_weight.float().expand(s["text"], 1, -1), w[s["text"]:]])
    y = y * w
    even, odd = y[..., 0::2], y[..., 1::2]
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    turned = torch.stack([even * cos[..., 0::2] - odd * sin[..., 0::2], odd * cos[..., 1::2] + even * sin[..., 1::2]], -1)
    return turned.flatten(-2).to(DTYPES[s["dtype"]])


def run(s):
    if own:
        return _own(s)
    if s["op"] == "qk":
        w = s["weights"]
        return (_rotated(s["q"], w["weight_q"], w.get("weight_txt_q"), s),
                _rotated(s["k"], w["weight_k"], w.get("weight_txt_k"), s))
    if s["op"] == "modulated":
        x = s["x"]
        if s["residual"]:
            x = (x.float() + s["gate"].float()[:, None] * s["y"].float()).to(x.dtype)
        f = x.float()
        f = f - f.mean(-1, keepdim=True)
        h = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)
        h = h * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
        out = _product(s, *_quantised(h))
        return (x, out) if s["residual"] else out
    if s["rows"] == "int8":
        return _product(s, s["codes"].float(), s["code_scales"][:, None])
    x = torch.cat([s["a"], s["b"]], dim=-1) if s["joined"] else s["x"]
    return _product(s, *_quantised(x.float()))


def work(case):
    """Each input read once, each output written once; 2 operations a product term."""
    if case["op"] == "qk":
        rows = case["batch"] * case["tokens"] * (case["hq"] + case["hk"])
        return {"bytes": rows * case["d"] * 4 + case["tokens"] * case["d"] * 4, "flops": rows * case["d"] * 10}
    k, n = case.get("k") or case["c"], case["n"]
    m = case.get("m") or case["batch"] * case["tokens"]
    moved = n * (k + 4) + m * n * 2 + (n * 2 if case.get("bias", True) else 0)
    if case["op"] == "modulated":
        moved += m * k * (6 if case["residual"] else 2) + case["batch"] * k * (6 if case["residual"] else 4)
    else:
        moved += m * (k + 4) if case["rows"] == "int8" else m * k * 2
    return {"bytes": moved, "flops": 2 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "qk":
        got = []
        for part in ("q", "k"):
            x = s[part].double()
            b, t, h, d = x.shape
            norm = x.square().sum(-1, keepdim=True).div(d).add(1e-6).sqrt()
            w = s["weights"]["weight_" + part].double().repeat(t, 1)
            if case["text"]:
                w[:case["text"]] = s["weights"]["weight_txt_" + part].double()
            z = torch.view_as_complex((x / norm * w[:, None]).view(b, t, h, d // 2, 2))
            turn = torch.complex(s["cos"][:, 0::2].double(), s["sin"][:, 0::2].double())
            got.append(torch.view_as_real(z * turn[:, None]).reshape(b, t, h, d))
        return tuple(got)
    stream = None
    if case["op"] == "modulated":
        x = s["x"].double()
        if case["residual"]:
            stream = torch.addcmul(x, s["gate"].double().unsqueeze(1), s["y"].double())
            x = stream.to(dt).double()  # the LayerNorm reads the stored stream
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        rows = torch.addcmul(s["shift"].double().unsqueeze(1), (x - mean) / (var + 1e-6).sqrt(),
                             s["scale"].double().unsqueeze(1) + 1)
    elif case["rows"] == "int8":
        rows = s["codes"].double() * s["code_scales"].double().unsqueeze(1)
    else:
        rows = torch.cat([s["a"], s["b"]], dim=1).double() if case["joined"] else s["x"].double()
    step = rows.abs().max(dim=-1, keepdim=True).values / 127
    if case.get("rows") != "int8":
        rows = (rows / step).round() * step
    out = torch.nn.functional.linear(rows, s["w"].double() * s["w_scales"].double().unsqueeze(1),
                                     None if s["bias_"] is None else s["bias_"].double())
    if case["act"]:
        u = math.sqrt(2 / math.pi) * (out + 0.044715 * out.pow(3))
        out = out / (1 + torch.exp(-2 * u))
    return out if stream is None else (stream, out)
