"""The operators beside the quantised cache whose speed is measured: rotary positions, the append that applies them, rows read
back out of the cache, and the linear attention of layers that keep a state instead of a cache.

A case names one call:

  rope    the position rotation of `tokens` rows of `heads` heads (queries and keys of one projection's output together)
  append  keys and values into the paged 4-bit cache of one layer, keys and queries rotated on the way; where the call completes
          tiles, these are read back, so that what the cache holds is among the outputs
  read    rows of one layer's cache back as 16-bit keys and values
  decode  linear attention with a decay for each head, one token of each of `batch` sequences
  chunk   the same over prompts: `batch` sequences packed one behind another, `tokens` in all

Geometries are the ones of this repository's workloads and tests (24 query heads over 4 key heads; 32 over 8, 16 over 2; heads of
128 or 256 dims, of which 64 turn at 256); linear layers have heads of 128 or 64 dims.  `run` computes them in elementary torch operations in
32 bits, or, with `own` set, by the framework's kernels; `exact` in 64 bits from the definitions.
"""
import math

import torch

own = False

PAGE, TILE = 64, 128
OUTLIERS = (3, 17, 64, 101)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _rope(name, tokens, start, heads, head_dim, rotary, dtype="fp16", layout="half", scaling="none", behind=0):
    return {"name": name, "op": "rope", "tokens": tokens, "start": start, "heads": heads, "head_dim": head_dim, "rotary": rotary, "dtype": dtype,
            "layout": layout, "scaling": scaling, "behind": behind}


def _append(name, tokens, start, kv_heads, q_heads, head_dim, rotary, dtype="fp16", layout="half", scaling="none"):
    return {"name": name, "op": "append", "tokens": tokens, "start": start, "kv_heads": kv_heads, "q_heads": q_heads, "head_dim": head_dim,
            "rotary": rotary, "dtype": dtype, "layout": layout, "scaling": scaling}


def _read(name, ctx, begin, tokens, kv_heads, head_dim, dtype="fp16"):
    return {"name": name, "op": "read", "ctx": ctx, "begin": begin, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype}


def _linear(name, op, batch, tokens, qk_heads, v_heads, head_dim, dtype="bf16"):
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "qk_heads": qk_heads, "v_heads": v_heads, "head_dim": head_dim, "dtype": dtype}


def listed():
    return [
        # one decode step in the engine's own geometry: a quarter of each head turns; latency alone
        _rope("rope_decode", 1, 30011, 28, 256, 64, dtype="bf16"),
        # a long prompt far into a scaled context: queries and keys of a fused projection, the values behind them in each row
        _rope("rope_prompt_8192", 8192, 131072, 28, 128, 128, scaling="yarn", behind=4),
        # one decode step: the newest token's key and value into the open tile, its queries turned beside it
        _append("append_decode", 1, 32768, 4, 24, 128, 128),
        # a short prompt of ragged length, neighbouring dims turned together
        _append("append_777", 777, 0, 4, 24, 128, 128, layout="interleaved"),
        # a chunk of an ordinary prompt in the engine's own geometry
        _append("append_1024_d256", 1024, 16384, 4, 24, 256, 64, dtype="bf16", scaling="linear"),
        # a prefix handed on to another engine, an odd range of it
        _read("read_5001_d256", 20000, 1003, 5001, 4, 256, dtype="bf16"),
        # a whole long context of one layer
        _read("read_131072", 131072, 0, 131072, 4, 128),
        # one user's decode step, one linear layer: the state of every head once over
        _linear("linear_decode", "decode", 1, 1, 16, 32, 128),
        # many users at once
        _linear("linear_decode_64", "decode", 64, 64, 16, 32, 128),
        # a short prompt of ragged length
        _linear("linear_300", "chunk", 1, 300, 16, 32, 128),
        # a long prompt
        _linear("linear_8192", "chunk", 1, 8192, 16, 32, 128),
        # several prompts of ragged lengths at once, fp16, the small head
        _linear("linear_batch_7", "chunk", 7, 9001, 24, 24, 64, dtype="fp16"),
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "append", "append", "read", "decode", "chunk", "chunk"))
    dtype, layout, scaling = rng.choice(("fp16", "bf16")), rng.choice(("half", "interleaved")), rng.choice(("none", "linear", "ntk", "yarn"))
    if op in ("decode", "chunk"):
        dim = rng.choice((64, 128, 128))
        qk, v = rng.choice(((16, 32), (16, 16), (8, 32), (24, 24), (4, 12), (1, 2)))
        if op == "decode":
            batch = _between(rng, 1, 64)
            c = _linear("", op, batch, batch, qk, v, dim, dtype)
        else:
            tokens = _between(rng, 20, min(16384, 8192 * 32 * 128 // (v * dim)))
            c = _linear("", op, rng.randint(1, min(12, tokens)), tokens, qk, v, dim, dtype)
    else:
        dim = rng.choice((128, 128, 256))
        kv, qh = rng.choice(((4, 24), (4, 24), (8, 32), (2, 16)))
        rotary = rng.choice((dim, dim, 64, 32, 96))
        if op == "rope":
            dim = rng.choice((dim, 64)) if rotary <= 64 else dim
            c = _rope("", _between(rng, 1, 8192 * 28 * 128 // ((kv + qh) * dim)), _between(rng, 1, 378944), kv + qh, dim, rotary, dtype, layout,
                      scaling, rng.choice((0, kv)))
        elif op == "append":
            tokens = _between(rng, 1, 2048)
            start = TILE * rng.randint(0, 256) if tokens > TILE else _between(rng, 1, 378000)
            c = _append("", tokens, start, kv, qh, dim, rotary, dtype, layout, scaling)
        else:
            ctx = _between(rng, 200, 131072 * 4 * 128 // (kv * dim))
            begin = rng.randint(0, ctx // 2)
            c = _read("", ctx, begin, rng.randint(1, ctx - begin), kv, dim, dtype)
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------------------


class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def table(self, pages):
        return torch.randperm(pages, generator=self.g, device="cuda").to(torch.int32)


def _with_outliers(x):
    """A few channels of every 128 are 20 times as large, as keys and values have them."""
    for s in range(0, x.shape[-1], 128):
        for ch in OUTLIERS:
            if s + ch < x.shape[-1]:
                x[..., s + ch] *= 20.0
    return x


_SCALING = {"none": {}, "linear": {"factor": 4.0}, "ntk": {"factor": 4.0}, "yarn": {"factor": 4.0, "original": 32768}}
_BASE = 1e6


def _frequencies(rotary, scaling, base=_BASE, beta_fast=32.0, beta_slow=1.0):
    """(radians a position of each pair, factor of cosine and sine)."""
    how = _SCALING[scaling]
    if scaling == "ntk" and rotary > 2:
        base = base * how["factor"] ** (rotary / (rotary - 2))
    freq = [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    if scaling == "linear":
        return [f / how["factor"] for f in freq], 1.0
    if scaling != "yarn":
        return freq, 1.0
    turns = lambda n: rotary * math.log(how["original"] / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(turns(beta_fast)), 0), min(math.ceil(turns(beta_slow)), rotary - 1)
    ramp = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(rotary // 2)]
    return [f / how["factor"] * r + f * (1 - r) for f, r in zip(freq, ramp)], 0.1 * math.log(how["factor"]) + 1.0


def _lengths(case):
    """Lengths of packed sequences: ragged, the longest about three times the shortest, `tokens` in all."""
    n, tokens = case["batch"], case["tokens"]
    share = [1 + (5 * i + 3) % n / max(1, n - 1) * 2 for i in range(n)]
    got = [max(1, int(tokens * s / sum(share))) for s in share]
    got[got.index(max(got))] += tokens - sum(got)
    return got


def _quantised(k, v, kv_heads, head_dim):
    """16-bit rotated rows [tiles * 128, heads, dims] of a cache as codes and axes: K's along the dims, V's along the tokens."""
    S = head_dim // 128
    x = k.view(-1, TILE, kv_heads, head_dim).float()
    lo, hi = x.amin(1, keepdim=True), x.amax(1, keepdim=True)
    step = ((hi - lo) / 15).clamp_min(1e-10)
    y = v.view(-1, TILE, kv_heads, S, 128).float()
    vlo, vhi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    vstep = ((vhi - vlo) / 15).clamp_min(1e-10)
    code = lambda a, b, s: ((a - b) / s + 0.5).floor().clamp(0, 15)  # noqa: E731
    return (code(x, lo, step), step.half(), lo.half()), (code(y, vlo, vstep), vstep.half(), vlo.half())


def _packed(codes):
    """Codes [pages, 64, heads, dims] -> bytes [pages, heads, 64, dims / 2]."""
    c = codes.to(torch.uint8).permute(0, 2, 1, 3)
    return (c[..., 0::2] | c[..., 1::2] << 4).contiguous()


def _planes(k, v, kv_heads, head_dim, table):
    """The four planes of a cache that holds the given rotated rows, pages in the table's order."""
    S, n = head_dim // 128, k.shape[0] // TILE
    (kc, ks, kz), (vc, vs, vz) = _quantised(k, v, kv_heads, head_dim)
    pages = table.numel()
    planes = [torch.zeros((pages, kv_heads, PAGE, w), dtype=t, device="cuda")
              for w, t in ((head_dim // 2, torch.uint8), (5 * S, torch.half), (head_dim // 2, torch.uint8), (4 * S, torch.half))]
    at = table[:2 * n].long()
    planes[0][at] = _packed(kc.view(2 * n, PAGE, kv_heads, head_dim))
    planes[2][at] = _packed(vc.view(2 * n, PAGE, kv_heads, head_dim))
    axis = lambda a: a.view(n, kv_heads, PAGE, 2 * S).repeat_interleave(2, 0)  # noqa: E731
    planes[1][at] = torch.cat((axis(ks), axis(kz), torch.ones((2 * n, kv_heads, PAGE, S), dtype=torch.half, device="cuda")), -1)
    token = lambda a: a.view(2 * n, PAGE, kv_heads, S).permute(0, 2, 1, 3)  # noqa: E731
    planes[3][at] = torch.cat((torch.ones((2 * n, kv_heads, PAGE, 2 * S), dtype=torch.half, device="cuda"), token(vs), token(vz)), -1)
    return planes


def _package():
    import __graft_entry__ as entry

    return entry.load_package()


def prepare(case, seed):
    gen, op, dtype = _Gen(seed), case["op"], DTYPES[case["dtype"]]
    state = {"case": case, "op": op}
    if op in ("decode", "chunk"):
        n, qk, vh, d = case["batch"], case["qk_heads"], case["v_heads"], case["head_dim"]
        rows = case["tokens"]
        state["q"], state["k"] = (gen.normal(rows, qk, d).to(dtype) for _ in range(2))
        state["v"] = gen.normal(rows, vh, d).to(dtype)
        # a state as such a sequence leaves it; sequences are read from the first half of the pool and written to the second
        log_decay = -torch.exp2(-8.0 * torch.arange(1, vh + 1, device="cuda") / vh)
        grown = (1 - torch.exp(2 * log_decay)).rsqrt()
        state["state"] = torch.cat((gen.normal(n, vh, d, d) * grown[None, :, None, None], torch.zeros((n, vh, d, d), device="cuda")))
        state["log_decay"], state["scale"] = log_decay, 1 / math.sqrt(d)
        order = torch.randperm(n, generator=gen.g, device="cuda").to(torch.int32)
        state["reads"], state["writes"] = order, torch.arange(n, 2 * n, dtype=torch.int32, device="cuda")
        if op == "chunk":
            lengths = _lengths(case)
            state["offsets"] = torch.tensor([sum(lengths[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda")
            state["longest"] = max(lengths)
        if own:
            state["layer"] = _package().LinearAttention(qk, vh, d, log_decay, 2 * n, dtype=dtype)
            state["layer"].state.copy_(state["state"])
            state["state"] = state["layer"].state
        return state
    if op == "read":
        kv, d, ctx = case["kv_heads"], case["head_dim"], case["ctx"]
        tiles = (ctx + TILE - 1) // TILE
        k, v = ((gen.normal(tiles * TILE, kv, d) * 4.5).half() for _ in range(2))
        state["table"] = gen.table(2 * tiles + 3)
        state["planes"] = _planes(k, v, kv, d, state["table"])
        stage = torch.zeros((2, 2, kv, TILE, d), dtype=torch.half, device="cuda")
        for i, x in enumerate((k, v)):  # the open tile's rows (or the last full one's), in its slot
            stage[i, (tiles - 1) % 2] = x[(tiles - 1) * TILE:].transpose(0, 1)
        state["stage"], state["pos"] = stage, torch.tensor([ctx - 1], dtype=torch.int32, device="cuda")
        if own:
            layer = _package().KvarnLayer(d, kv, kv, state["table"].numel(), state["table"], dtype=dtype)
            for mine, x in zip((layer.k_code, layer.k_scale, layer.v_code, layer.v_scale), state["planes"]):
                mine.copy_(x)
            layer.stage.copy_(stage.view(-1))
            state["layer"] = layer
        return state
    d, tokens = case["head_dim"], case["tokens"]
    freq, state["factor"] = _frequencies(case["rotary"], case["scaling"])
    state["freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
    state["pos"] = torch.arange(case["start"], case["start"] + tokens, dtype=torch.int32, device="cuda")
    if own:
        state["rope"] = _package().Rope(case["rotary"], base=_BASE, scaling=case["scaling"], interleaved=case["layout"] == "interleaved",
                                        **_SCALING[case["scaling"]])
    if op == "rope":
        fused = _with_outliers(gen.normal(tokens, case["heads"] + case["behind"], d)).to(dtype)
        state["x"] = fused[:, :case["heads"]]
        return state
    kv, qh = case["kv_heads"], case["q_heads"]
    state["q"] = gen.normal(tokens, qh, d).to(dtype)
    state["k"], state["v"] = (_with_outliers(gen.normal(tokens, kv, d)).to(dtype) for _ in range(2))
    state["stage"] = torch.zeros((2, 2, kv, TILE, d), dtype=torch.half, device="cuda")
    live = case["start"] % TILE  # rows that earlier calls left in the open tile
    state["stage"][:, case["start"] // TILE % 2, :, :live] = (gen.normal(2, kv, live, d) * 4.5).half()
    tiles = (case["start"] + tokens + TILE - 1) // TILE
    state["table"] = gen.table(2 * tiles + 2)
    state["sealed"] = (case["start"] + tokens) // TILE - case["start"] // TILE  # tiles that the call completes
    if own:
        layer = _package().KvarnLayer(d, kv, qh, state["table"].numel(), state["table"], dtype=dtype)
        layer.stage.copy_(state["stage"].view(-1))
        state["layer"] = layer
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------------------


def _hadamard(n, dtype=torch.float32):
    """The Sylvester matrix by the parity of the common bits of row and column, normalised."""
    i = torch.arange(n, device="cuda")
    both = i[:, None] & i[None, :]
    for_bits = torch.arange(n.bit_length() - 1, device="cuda")
    odd = (both[..., None] >> for_bits & 1).sum(-1) & 1
    return (1 - 2 * odd).to(dtype) / math.sqrt(n)


def _turned(x, pos, freq, factor, rotary, layout, wide=torch.float32):
    """Rows x [tokens, heads, dims] with their first `rotary` dims turned by the positions' angles."""
    angle = pos.double()[:, None] * freq
    c, s = ((f(angle) * factor).to(wide)[:, None] for f in (torch.cos, torch.sin))
    x = x.to(wide)
    if layout == "half":
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        return torch.cat((a * c - b * s, b * c + a * s, x[..., rotary:]), -1)
    a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    return torch.cat((torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), x[..., rotary:]), -1)


def _plain_append(st):
    c, pos = st["case"], st["pos"]
    dtype, d, kv, tokens, start = DTYPES[c["dtype"]], c["head_dim"], c["kv_heads"], c["tokens"], c["start"]
    H = _hadamard(d)
    q = _turned(st["q"], pos, st["freq"], st["factor"], c["rotary"], c["layout"]).to(dtype)
    rows = [(_turned(st["k"], pos, st["freq"], st["factor"], c["rotary"], c["layout"]) @ H).half(), (st["v"].float() @ H).half()]
    # the stage keeps the rows of the last two tiles, each in its slot
    stage, first = st["stage"].clone(), max(start, ((start + tokens - 1) // TILE - 1) * TILE)
    at = torch.arange(first, start + tokens, device="cuda")
    stage[0, at // TILE % 2, :, at % TILE], stage[1, at // TILE % 2, :, at % TILE] = rows[0][first - start:], rows[1][first - start:]
    if not st["sealed"]:
        return {"q": q, "stage": stage}
    base = start // TILE * TILE
    before = [st["stage"][i, start // TILE % 2, :, :start - base].transpose(0, 1) for i in range(2)]
    whole = st["sealed"] * TILE
    k, v = (torch.cat((b, r))[:whole] for b, r in zip(before, rows))
    (kc, ks, kz), (vc, vs, vz) = _quantised(k, v, kv, d)
    k, v = ((a * b.float() + z.float()).reshape(whole, kv, d) @ H for a, b, z in ((kc, ks, kz), (vc, vs, vz)))
    return {"q": q, "stage": stage, "k": k.to(dtype), "v": v.to(dtype)}


def _plain_read(st):
    c = st["case"]
    d, kv, begin, end, dtype = c["head_dim"], c["kv_heads"], c["begin"], c["begin"] + c["tokens"], DTYPES[c["dtype"]]
    S, sealed, H = d // 128, c["ctx"] // TILE * TILE, _hadamard(d)
    k_code, k_scale, v_code, v_scale = st["planes"]
    at = torch.arange(begin, min(end, sealed), device="cuda")
    page, row, dim = st["table"].long()[at // PAGE], at % PAGE, torch.arange(d, device="cuda")
    unpack = lambda b: torch.stack((b & 15, b >> 4), -1).flatten(-2).float()  # noqa: E731
    per_dim = lambda plane, col: plane[..., col:col + 2 * S].reshape(plane.shape[0], kv, d)[page].float()  # noqa: E731
    per_token = lambda plane, col: plane[page, :, row, col:col + S].float().repeat_interleave(128, -1)  # noqa: E731
    k = (unpack(k_code[page, :, row]) * per_dim(k_scale, 0) + per_dim(k_scale, 2 * S)) * per_token(k_scale, 4 * S)
    v = (unpack(v_code[page, :, row]) * per_token(v_scale, 2 * S) + per_token(v_scale, 3 * S)) * per_dim(v_scale, 0)
    if end > sealed:
        open_rows = st["stage"][:, sealed // TILE % 2, :, max(begin, sealed) - sealed:end - sealed].transpose(1, 2).float()
        k, v = torch.cat((k, open_rows[0])), torch.cat((v, open_rows[1]))
    return {"k": (k @ H).to(dtype), "v": (v @ H).to(dtype)}


def _plain_decode(st):
    c = st["case"]
    share = c["v_heads"] // c["qk_heads"]
    q, k = (x.float().repeat_interleave(share, 1) for x in (st["q"], st["k"]))
    new = st["state"][st["reads"].long()] * torch.exp(st["log_decay"])[None, :, None, None] + k[..., :, None] * st["v"].float()[..., None, :]
    out = (q[..., None, :] @ new)[..., 0, :] * st["scale"]
    return {"out": out.to(DTYPES[c["dtype"]]), "state": new}


def _plain_chunk(st, C=64):
    """Sequences padded to chunks of C: products inside a chunk, and the chunks' own sums carried over by one product with their decays."""
    c = st["case"]
    d, vh, n = c["head_dim"], c["v_heads"], c["batch"]
    share, blocks = vh // c["qk_heads"], (st["longest"] + C - 1) // C
    begin, length = st["offsets"][:-1].long(), (st["offsets"][1:] - st["offsets"][:-1]).long()
    at = torch.arange(blocks * C, device="cuda")
    valid = at[None] < length[:, None]
    index = (begin[:, None] + at[None]).clamp_max(c["tokens"] - 1)
    pick = lambda x, r: (x.float()[index] * valid[..., None, None]).repeat_interleave(r, 2).transpose(1, 2).reshape(n, vh, blocks, C, d)  # noqa: E731
    q, k, v = pick(st["q"], share), pick(st["k"], share), pick(st["v"], 1)
    g, i = st["log_decay"], torch.arange(C, device="cuda")
    gap = i[:, None] - i[None, :]
    inside = torch.where(gap >= 0, torch.exp(g[:, None, None] * gap.clamp_min(0)), 0.0)[:, None]
    out = ((q @ k.transpose(-1, -2)) * inside) @ v
    sums = (k * torch.exp(g[:, None] * (C - 1 - i))[:, None, :, None]).transpose(-1, -2) @ v
    b = torch.arange(blocks, device="cuda")
    gap = b[:, None] - 1 - b[None, :]
    over = torch.where(gap >= 0, torch.exp(g[:, None, None] * C * gap.clamp_min(0)), 0.0)
    first = st["state"][st["reads"].long()]
    carried = (over @ sums.reshape(n, vh, blocks, d * d)).reshape(n, vh, blocks, d, d) + first[:, :, None] * torch.exp(g[:, None] * C * b)[..., None, None]
    out = out + (q @ carried) * torch.exp(g[:, None] * (i + 1))[:, None, :, None]
    out = (out * st["scale"]).reshape(n, vh, blocks * C, d).transpose(1, 2)[valid]
    left = torch.exp(g[None, :, None] * (length[:, None] - 1 - at[None]).clamp_min(0)[:, None])[..., None]
    new = (k.reshape(n, vh, -1, d) * left).transpose(-1, -2) @ v.reshape(n, vh, -1, d) + first * torch.exp(g[None] * length[:, None])[..., None, None]
    return {"out": out.to(DTYPES[c["dtype"]]), "state": new}


def run(state):
    op, c = state["op"], state["case"]
    if not own:
        if op == "rope":
            return _turned(state["x"], state["pos"], state["freq"], state["factor"], c["rotary"], c["layout"]).to(DTYPES[c["dtype"]])
        return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "chunk": _plain_chunk}[op](state)
    if op == "rope":
        return state["rope"].rows(state["x"], state["pos"])
    layer = state["layer"]
    if op == "append":
        q = layer.rope_append(state["rope"], state["k"], state["v"], state["pos"], q=state["q"])
        stage = layer.stage.view(state["stage"].shape)
        if not state["sealed"]:
            return {"q": q, "stage": stage}
        k, v = layer.read_rows(c["start"] // TILE * TILE, state["sealed"] * TILE, state["pos"][-1:])
        return {"q": q, "stage": stage, "k": k, "v": v}
    if op == "read":
        k, v = layer.read_rows(c["begin"], c["tokens"], state["pos"])
        return {"k": k, "v": v}
    if op == "decode":
        out = layer.decode(state["q"], state["k"], state["v"], state["scale"], state["reads"], state["writes"])
    else:
        out = layer.chunk(state["q"], state["k"], state["v"], state["offsets"], state["scale"], state["reads"], state["writes"])
    return {"out": out, "state": layer.state[c["batch"]:]}  # the pool's second half, as the sequences wrote it


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------


def work(case):
    op, d = case["op"], case["head_dim"]
    if op == "rope":
        return {"bytes": case["tokens"] * (4 * case["heads"] * d + 4), "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    if op == "append":
        tokens, kv, qh, S = case["tokens"], case["kv_heads"], case["q_heads"], d // 128
        last = case["start"] + tokens
        sealed = last // TILE - case["start"] // TILE
        staged = last - max(case["start"], ((last - 1) // TILE - 1) * TILE)
        old = case["start"] % TILE if sealed else 0
        rows = tokens * (4 * qh * d + 4 * kv * d + 4)  # queries in and out, keys and values in
        held = sealed * TILE * kv * (d + 12 * S + 4 * d)  # the tiles' codes and axes, and their values as they are read back
        return {"bytes": rows + (staged + old) * 4 * kv * d + held, "flops": 3 * tokens * (qh + kv) * case["rotary"] + 2 * (tokens + sealed * TILE) * kv * d * int(math.log2(d))}
    if op == "read":
        kv, begin, end, sealed = case["kv_heads"], case["begin"], case["begin"] + case["tokens"], case["ctx"] // TILE * TILE
        coded = max(0, min(end, sealed) - begin)
        return {"bytes": kv * (coded * (d + 12 * (d // 128)) + (case["tokens"] - coded) * 4 * d + case["tokens"] * 4 * d), "flops": 2 * case["tokens"] * kv * d * (int(math.log2(d)) + 2)}
    qk, vh, n, tokens = case["qk_heads"], case["v_heads"], case["batch"], case["tokens"]
    rows = tokens * 2 * d * (2 * qk + 2 * vh)
    states = n * vh * d * d * 8
    # a token's outer product, decay and product with the query
    return {"bytes": rows + states, "flops": 5 * tokens * vh * d * d}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------


def _exact_turned(x, case, pos):
    """Each pair as a complex number, times factor * exp(i position frequency)."""
    r = case["rotary"]
    freq, factor = _frequencies(r, case["scaling"])
    x = x.double().clone()
    turn = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda"), pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device="cuda"))
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_wht(x):
    """Walsh-Hadamard along the last axis by its recursion on halves."""
    n = x.shape[-1]
    span = 1
    while span < n:
        y = x.reshape(*x.shape[:-1], n // (2 * span), 2, span)
        x = torch.stack((y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]), -2).reshape(*x.shape)
        span *= 2
    return x / math.sqrt(n)


def _exact_held(matrix):
    """Rows of 16-bit values -> what 4-bit codes with a 16-bit step and zero point along each stand for.  Which code a value gets is defined
    by the cache's format, whose step and quotient are 32-bit numbers: 16-bit values meet the middle between two codes often."""
    x = matrix.float()
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    step = torch.maximum((hi - lo) / 15, torch.full_like(hi, 1e-10))
    code = torch.clamp(torch.floor(((x - lo) / step).double() + 0.5), 0, 15)
    return code * step.half().double() + lo.double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op, d = case["op"], case["head_dim"]
    if op == "rope":
        return _exact_turned(st["x"], case, st["pos"])
    if op == "append":
        out = {"q": _exact_turned(st["q"], case, st["pos"])}
        k, v = _exact_wht(_exact_turned(st["k"], case, st["pos"])).half().double(), _exact_wht(st["v"].double()).half().double()
        tokens, start, kv = case["tokens"], case["start"], case["kv_heads"]
        stage = st["stage"].double().clone()
        last_tile = (start + tokens - 1) // TILE
        held = {"k": [], "v": []}
        for tile in range(start // TILE, last_tile + 1):
            lo, hi = max(start, tile * TILE), min(start + tokens, (tile + 1) * TILE)
            rows = st["stage"][:, tile % 2].double().clone()  # [2, heads, 128, dims]: rows of earlier calls, then the new ones
            for which, x in enumerate((k, v)):
                rows[which, :, lo - tile * TILE:hi - tile * TILE] = x[lo - start:hi - start].transpose(0, 1)
            if hi == (tile + 1) * TILE:
                held["k"].append(_exact_wht(_exact_held(rows[0].transpose(1, 2)).transpose(1, 2)).transpose(0, 1))
                held["v"].append(_exact_wht(_exact_held(rows[1].reshape(kv, TILE, d // 128, 128)).reshape(kv, TILE, d)).transpose(0, 1))
            if tile >= last_tile - 1:
                stage[:, tile % 2, :, lo - tile * TILE:hi - tile * TILE] = rows[:, :, lo - tile * TILE:hi - tile * TILE]
        out["stage"] = stage
        if held["k"]:
            out.update({name: torch.cat(x) for name, x in held.items()})
        return out
    if op == "read":
        kv, begin, end, S = case["kv_heads"], case["begin"], case["begin"] + case["tokens"], d // 128
        out = [], []
        for tile in range(begin // TILE, (end - 1) // TILE + 1):
            if (tile + 1) * TILE <= case["ctx"]:
                k_code, k_scale, v_code, v_scale = (torch.cat([p[int(st["table"][2 * tile + i])] for i in range(2)], 1) for p in st["planes"])
                ks, vs, one = k_scale.double(), v_scale.double(), PAGE
                codes = [torch.stack((c & 15, c >> 4), -1).reshape(kv, TILE, d).double() for c in (k_code, v_code)]
                k = codes[0] * ks[:, :one, :2 * S].reshape(kv, 1, d) + ks[:, :one, 2 * S:4 * S].reshape(kv, 1, d)
                k = (k.reshape(kv, TILE, S, 128) * ks[:, :, 4 * S:, None]).reshape(kv, TILE, d)
                v = codes[1].reshape(kv, TILE, S, 128) * vs[:, :, 2 * S:3 * S, None] + vs[:, :, 3 * S:, None]
                v = v.reshape(kv, TILE, d) * vs[:, :one, :2 * S].reshape(kv, 1, d)
            else:
                k, v = st["stage"][:, tile % 2].double()
            lo, hi = max(begin - tile * TILE, 0), min(end - tile * TILE, TILE)
            for to, x in zip(out, (k, v)):
                to.append(_exact_wht(x[:, lo:hi]).transpose(0, 1))
        return {"k": torch.cat(out[0]), "v": torch.cat(out[1])}
    n, qk, vh = case["batch"], case["qk_heads"], case["v_heads"]
    lengths = _lengths(case) if op == "chunk" else [1] * n
    out, states, at = [], [], 0
    for b, length in enumerate(lengths):
        rows = slice(at, at + length)
        at += length
        per_head, new = [], []
        t = torch.arange(length, device="cuda", dtype=torch.float64)
        for h in range(vh):
            q, k, v = st["q"][rows, h * qk // vh].double(), st["k"][rows, h * qk // vh].double(), st["v"][rows, h].double()
            first, g = st["state"][int(st["reads"][b]), h].double(), st["log_decay"][h].double()
            seen = (torch.exp(g * (t[:, None] - t[None, :]).clamp_min(0)) * (q @ k.T)).tril()
            per_head.append((seen @ v + torch.exp(g * (t + 1))[:, None] * (q @ first)) * st["scale"])
            new.append(torch.exp(g * length) * first + (k * torch.exp(g * (length - 1 - t))[:, None]).T @ v)
        out.append(torch.stack(per_head, 1))
        states.append(torch.stack(new))
    return {"out": torch.cat(out), "state": torch.stack(states)}
