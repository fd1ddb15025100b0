"""The 8-bit paged KV cache (written, read back, attended over) and rotary positions with several axes, as cases that can be
timed and compared: in plain torch operations (`own` false) and through this package's public objects (`own` true).

A cached row is one token of one kv head, D elements x.  Its step is 2^e, e the smallest whole number, at least -126, with
max |x| < 127.5 * 2^e; it is held as whole numbers rint(x / 2^e) from -127 to 127 and one byte e + 127."""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
PAGE = 16


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # A server's decode step: 64 sequences of 1024 to 8192 tokens in permuted 16-token pages.
        {"name": "decode8_batch", "kind": "decode", "B": 64, "Hq": 32, "Hkv": 8, "D": 128, "lo": 1024, "hi": 8192, "dtype": "bf16", "out": "f32"},
        # One sequence of 131072 tokens, 64 query heads.
        {"name": "decode8_long", "kind": "decode", "B": 1, "Hq": 64, "Hkv": 8, "D": 128, "lo": 131072, "hi": 131072, "dtype": "bf16", "out": "bf16"},
        # One user's next token over a short conversation: the smallest decode.
        {"name": "decode8_chat", "kind": "decode", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "lo": 1411, "hi": 1411, "dtype": "bf16", "out": "bf16"},
        # A small model's batch: head_dim 64, f32 activations, very ragged, some sequences of a few tokens.
        {"name": "decode8_ragged64", "kind": "decode", "B": 24, "Hq": 14, "Hkv": 2, "D": 64, "lo": 3, "hi": 2500, "dtype": "f32", "out": "f32"},
        # A batch of full prompts written and read back for the layer's own attention over them.
        {"name": "write8_batch", "kind": "write", "B": 4, "Hkv": 8, "D": 128, "past": 0, "n": 4096, "dtype": "bf16", "out": "bf16"},
        # A follow-up of an odd length from f32 activations on a warm cache: its rows written, all rows read back.
        {"name": "write8_follow", "kind": "write", "B": 1, "Hkv": 8, "D": 128, "past": 1311, "n": 201, "dtype": "f32", "out": "bf16"},
        # One new token of 16 short sequences: the smallest write.
        {"name": "write8_token", "kind": "write", "B": 16, "Hkv": 2, "D": 64, "past": 30, "n": 1, "dtype": "bf16", "out": "f32"},
        # RoPE of q and k with the quantising append, for the batch of prompts.
        {"name": "rotate8_batch", "kind": "rotate", "B": 4, "Hq": 32, "Hkv": 8, "D": 128, "n": 4096, "dtype": "bf16", "interleaved": False},
        # One chat prompt of an odd length, adjacent pairs, from f32 activations.
        {"name": "rotate8_prompt", "kind": "rotate", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "n": 777, "dtype": "f32", "interleaved": True},
        # The patches of one image in an image tower: rows and columns as two axes, head_dim 80, q and k alone.
        {"name": "axes_image", "kind": "axes", "B": 1, "Hq": 16, "Hkv": 16, "D": 80, "sections": "20,20", "pages": "", "rows": 58, "cols": 74,
         "before": 0, "after": 0, "dtype": "f32", "interleaved": False},
        # A prompt with a picture in it: time, height and width, rotated and written to the 16-bit cache.
        {"name": "axes_prompt", "kind": "axes", "B": 1, "Hq": 28, "Hkv": 4, "D": 128, "sections": "16,24,24", "pages": "bf16", "rows": 38, "cols": 51,
         "before": 23, "after": 96, "dtype": "bf16", "interleaved": False},
        # A batch of such prompts written to the 8-bit cache.
        {"name": "axes8_batch", "kind": "axes", "B": 4, "Hq": 32, "Hkv": 8, "D": 128, "sections": "16,24,24", "pages": "i8", "rows": 60, "cols": 60,
         "before": 300, "after": 196, "dtype": "bf16", "interleaved": False},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most=64):
    while True:
        hkv, g = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 3, 4, 4, 5, 7, 8))
        if hkv * g <= most:
            return hkv * g, hkv


def draw(rng):
    kind = rng.choice(("decode", "decode", "decode", "write", "write", "rotate", "axes", "axes"))
    D = rng.choice((128, 128, 64))
    Hq, Hkv = _heads(rng)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "decode":
        hi = _log(rng, 1, 131072)
        B = _log(rng, 1, max(1, min(128, (1 << 28) // (Hkv * D * hi))))
        return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "lo": max(1, int(hi * rng.uniform(0.02, 1.0))), "hi": hi, "dtype": dtype,
                "out": rng.choice(("f32", "bf16", "f16"))}
    B = rng.choice((1, 1, 2, 4, 16))
    most = (1 << 26) // (B * (Hq + 2 * Hkv) * D)  # tokens of a sequence
    if kind == "write":
        n = _log(rng, 1, max(2, (1 << 24) // (B * Hkv * D)))
        return {"kind": kind, "B": B, "Hkv": Hkv, "D": D, "past": _log(rng, 1, 2 * n + 64) if rng.random() < 0.4 else 0, "n": n, "dtype": dtype,
                "out": rng.choice(("bf16", "f32", "f16"))}
    if kind == "rotate":
        return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "n": _log(rng, 1, max(2, most)), "dtype": dtype, "interleaved": rng.random() < 0.4}
    pages = rng.choice(("", "bf16", "i8", "i8"))
    D = rng.choice((64, 80, 96, 128)) if pages == "" else D
    half = D // 2
    if rng.random() < 0.4:
        a = rng.choice((half // 2, half // 4))
        sections = (a, half - a)
    else:
        a = rng.choice((half // 4, half // 3))
        sections = (a, (half - a) // 2, half - a - (half - a) // 2)
    rows, cols = _log(rng, 1, 48), _log(rng, 1, 64)
    while rows * cols > max(2, most // 2):
        rows, cols = max(1, rows // 2), max(1, cols // 2)
    return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "sections": ",".join(map(str, sections)), "pages": pages, "rows": rows, "cols": cols,
            "before": rng.choice((0, 5, _log(rng, 1, max(2, most // 4)))), "after": rng.choice((0, 9, _log(rng, 1, max(2, most // 4)))), "dtype": dtype,
            "interleaved": rng.random() < 0.3}


# ------------------------------------------------------------------------------------------------------------ inputs
def _lengths(c):
    """The sequence lengths of a decode batch: evenly from lo to hi."""
    B, lo, hi = c["B"], c["lo"], c["hi"]
    return [hi if B == 1 else lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _tokens(c):
    return c["n"] if "n" in c else c["before"] + c["rows"] * c["cols"] + c["after"]


def _axis_of_pair(c):
    """The axis of each pair: the sections in order."""
    return [a for a, n in enumerate(c["sections"].split(",")) for _ in range(int(n))]


def _pick(c):
    """The axis of each pair as an index on the GPU."""
    return torch.tensor(_axis_of_pair(c), device="cuda")


def _positions(c):
    """[axes, B, tokens]: text counts on along every axis, the picture's tokens stand at their row and column (and one time)."""
    axes = len(c["sections"].split(","))
    grid = torch.stack(torch.meshgrid(torch.arange(c["rows"]), torch.arange(c["cols"]), indexing="ij")).reshape(2, -1)
    if axes == 3:
        grid = torch.cat([torch.zeros_like(grid[:1]), grid])
    start, end = c["before"], c["before"] + max(c["rows"], c["cols"])
    one = torch.cat([torch.arange(start).expand(axes, -1), grid + start, end + torch.arange(c["after"]).expand(axes, -1)], 1)
    shift = 3 * torch.arange(c["B"])  # the sequences of a batch do not start at the same place
    return (one[:, None] + shift[:, None]).to(torch.int32).cuda()


def _tables(c, rows):
    half = c["D"] // 2
    # with two axes both halves of the pairs have the same frequencies
    period = half if c.get("sections", "").count(",") != 1 else int(c["sections"].split(",")[0])
    inv = 10000.0 ** (-(torch.arange(half, device="cuda", dtype=torch.float64) % period) / period)
    ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _rows_of(c, gen, shape, dtype):
    """Keys or values: normal, with a few channels several times as large and a token in fifty small."""
    x = torch.randn(shape, generator=gen, device="cuda")
    big = torch.rand(shape[1:2] + (1,) + shape[3:], generator=gen, device="cuda") < 0.03
    small = torch.rand(shape[:-1] + (1,), generator=gen, device="cuda") < 0.02
    return (x * torch.where(big, 6.0, 1.0) * torch.where(small, 0.01, 1.0)).to(TORCH[dtype])


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    B, Hkv, D, dt = c["B"], c["Hkv"], c["D"], TORCH[c["dtype"]]
    s = {"case": c}
    if c["kind"] == "decode":
        host = torch.Generator().manual_seed(int(seed))
        lens = torch.tensor(_lengths(c))[torch.randperm(B, generator=host)]
        pages = (lens + PAGE - 1) // PAGE
        total, widest = int(pages.sum()), int(pages.max())
        order, at = torch.randperm(total, generator=host), torch.cumsum(pages, 0) - pages
        slot = torch.arange(widest)[None]
        table = torch.where(slot < pages[:, None], order[(at[:, None] + slot).clamp(max=total - 1)], 0)
        codes = [torch.empty((total, Hkv, PAGE, D), device="cuda", dtype=torch.int8) for _ in range(2)]
        scales = torch.empty((total, Hkv, 2, PAGE), device="cuda", dtype=torch.uint8)
        for which in range(2):
            for i in range(0, total, 4096):
                held, e = _quantise(_rows_of(c, gen, (min(4096, total - i), Hkv, PAGE, D), "bf16").float())
                codes[which][i:i + 4096], scales[i:i + 4096, :, which] = held.to(torch.int8), (e + 127).to(torch.uint8)
        s.update(k=codes[0], v=codes[1], scales=scales, table=table.cuda(), lens=lens.cuda(), lens_host=lens, table_host=table, scale=D ** -0.5,
                 q=torch.randn((B, c["Hq"], 1, D), generator=gen, device="cuda").to(dt))
    else:
        n = _tokens(c)
        s.update(k=_rows_of(c, gen, (B, Hkv, n, D), c["dtype"]), v=_rows_of(c, gen, (B, Hkv, n, D), c["dtype"]))
        if c["kind"] == "write":
            s.update(k0=_rows_of(c, gen, (B, Hkv, c["past"], D), c["dtype"]), v0=_rows_of(c, gen, (B, Hkv, c["past"], D), c["dtype"]))
        else:
            s["q"] = torch.randn((B, c["Hq"], n, D), generator=gen, device="cuda").to(dt)
            if c["kind"] == "axes":
                s.update(positions=_positions(c), axis=_pick(c))
            s["cos"], s["sin"] = _tables(c, int(s["positions"].max()) + 1 if c["kind"] == "axes" else n)
    if own:
        _hold(s)
    return s


# ------------------------------------------------------------------------------------------------------------ the plain form
def _power(e):
    """2^e in f32, e a whole number from -126 to 127."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """f32 rows [..., D] -> the whole numbers of each row as f32, and its exponent e [...]."""
    m, e = torch.frexp(x.abs().amax(-1))  # max |x| = m * 2^e, m from 1/2 up to 1, or 0
    e = torch.where(m < 127.5 / 128, e - 7, e - 6).clamp(min=-126)
    return torch.round(x * _power(-e)[..., None]), e


def _held(x):
    """What the 8-bit cache holds of f32 rows, as values."""
    code, e = _quantise(x)
    return code * _power(e)[..., None]


def _rotate(x, cos, sin, interleaved):
    """x [B, H, n, D] in f32, cos and sin [B or 1, n, D / 2]."""
    cos, sin, half = cos[:, None], sin[:, None], x.shape[-1] // 2
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos + (-b) * sin, b * cos + a * sin], -1)


def _plain_decode(s):
    c, table = s["case"], s["table"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]

    def rows(which, codes):
        values = codes[table].float() * _power(s["scales"][table][:, :, :, which].to(torch.int32) - 127)[..., None]
        return values.transpose(1, 2).reshape(B, Hkv, -1, D)

    scores = s["q"].float().view(B, Hkv, Hq // Hkv, D) @ rows(0, s["k"]).transpose(-1, -2) * s["scale"]
    there = torch.arange(scores.shape[-1], device="cuda") < s["lens"][:, None]
    scores = torch.where(there[:, None, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = p @ rows(1, s["v"]) / p.sum(-1, keepdim=True)
    return out.view(B, Hq, 1, D).to(TORCH[c["out"]])


def _angles(s):
    """cos and sin of every token and pair, [B or 1, n, D / 2]."""
    c = s["case"]
    if c["kind"] == "rotate":
        return s["cos"][None], s["sin"][None]
    row = s["positions"].long()[s["axis"]].permute(1, 2, 0)  # [B, n, D / 2]
    return s["cos"].gather(0, row.flatten(0, 1)).view(row.shape), s["sin"].gather(0, row.flatten(0, 1)).view(row.shape)


def run(state):
    s, c = state, state["case"]
    if own:
        return _own_run(s)
    if c["kind"] == "decode":
        return _plain_decode(s)
    if c["kind"] == "write":
        return tuple(_held(torch.cat([s[x + "0"], s[x]], 2).float()).to(TORCH[c["out"]]) for x in "kv")
    cos, sin = _angles(s)
    q, k = (_rotate(s[x].float(), cos, sin, c["interleaved"]) for x in "qk")
    q = q.to(s["q"].dtype)
    if c["kind"] == "axes" and c["pages"] == "":
        return q, k.to(s["k"].dtype)
    if c["kind"] == "axes" and c["pages"] == "bf16":
        return q, k.to(torch.bfloat16), s["v"].to(torch.bfloat16)
    return q, _held(k).to(torch.bfloat16), _held(s["v"].float()).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------------------ the package's calls
_dev = None


def _device():
    """One library context for the life of the process, on torch's stream, as a program has it that does the rest in torch."""
    global _dev
    if _dev is None:
        import floneum_b200 as fb
        _dev = fb.Device.gpu(0)
        _dev.set_stream(torch.cuda.current_stream().cuda_stream)
    return _dev


class _Borrowed:
    """A library tensor (or a raw device pointer) in the form torch can wrap without a copy."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "typestr": typestr, "strides": None, "version": 3}


def _torch(t):
    """The library's result as a torch tensor on the same memory."""
    x = torch.as_tensor(_Borrowed(t, t.ptr, t.shape(), "<f4" if t.dtype == 0 else "<i2"), device="cuda")
    return x if t.dtype == 0 else x.view(torch.bfloat16 if t.dtype == 1 else torch.float16)


def _hold(s):
    """The library's objects of a state: tensors on the same memory, and the cache as the steps before have left it."""
    import floneum_b200 as fb
    c, dev = s["case"], _device()
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    s["t"] = t = {x: fb.Tensor.from_torch(dev, s[x]) for x in ("q", "k", "v", "k0", "v0", "cos", "sin", "positions") if x in s and (c["kind"], x) not in
                  (("decode", "k"), ("decode", "v"))}
    if c["kind"] == "decode":
        s["cache"] = cache = fb.PagedKvCache(dev, B, Hkv, D, s["k"].shape[0], s["table"].shape[1], dtype=fb.I8)
        for ptr, x, typestr in zip(cache.pools() + (cache.scales(),), (s["k"], s["v"], s["scales"]), ("|i1", "|i1", "|u1")):
            torch.as_tensor(_Borrowed(cache, ptr, tuple(x.shape), typestr), device="cuda").copy_(x)
        cache.set_page_table(s["table_host"].to(torch.int32).numpy(), s["lens_host"].to(torch.int32).numpy())
        s["answer"] = torch.empty((B, c["Hq"], 1, D), device="cuda", dtype=TORCH[c["out"]])
        t["answer"] = fb.Tensor.from_torch(dev, s["answer"])
        return
    if c["kind"] == "axes":
        s["axes"] = fb.axes_of_sections([int(x) for x in c["sections"].split(",")])
    if c["kind"] != "write":
        s["rope"] = fb.RopeCache.from_parts(t["cos"], t["sin"])
    past = c.get("past", 0)
    pages = (past + _tokens(c) + PAGE - 1) // PAGE
    s["cache"] = cache = fb.PagedKvCache(dev, B, Hkv, D, B * pages, pages, dtype=fb.BF16 if c.get("pages") == "bf16" else fb.I8) if D in (64, 128) else None
    if past:
        used = (past + PAGE - 1) // PAGE
        cache.append(t["k0"], t["v0"])  # a new cache hands its pages out in order, sequence after sequence
        s["table_host"] = (torch.arange(B)[:, None] * used + torch.arange(pages)[None].clamp(max=used - 1)).to(torch.int32).numpy()
        s["past_host"] = torch.full((B,), past, dtype=torch.int32).numpy()


def _own_run(s):
    c, t, cache = s["case"], s["t"], s["cache"]
    if c["kind"] == "decode":
        cache.decode(t["q"], s["scale"], t["answer"])
        return s["answer"]
    if c["kind"] == "write":
        if c["past"]:
            cache.set_page_table(s["table_host"], s["past_host"])  # the scheduler says what the batch is at every step
        else:
            cache.reset()
        cache.append(t["k"], t["v"])
        k, v = cache.gather(c["B"], c["past"] + c["n"], {"f32": 0, "bf16": 1, "f16": 2}[c["out"]])
        return _torch(k), _torch(v)
    where = dict(positions=t["positions"], axes=s["axes"]) if c["kind"] == "axes" else dict(start_pos=0)
    if c.get("pages") == "":
        q, k = s["rope"].forward_axes(t["q"], t["k"], interleaved=c["interleaved"], **where)
        return _torch(q), _torch(k)
    cache.reset()
    q = s["rope"].forward_append(t["q"], t["k"], t["v"], cache, interleaved=c["interleaved"], **where)
    k, v = cache.gather(c["B"], _tokens(c), 1)
    return _torch(q), _torch(k), _torch(v)


# ------------------------------------------------------------------------------------------------------------ what it takes
def work(case):
    c = case
    B, Hkv, D, e = c["B"], c["Hkv"], c["D"], SIZE[c["dtype"]]
    if c["kind"] == "decode":
        tokens = sum(_lengths(c))
        return {"bytes": 2.0 * Hkv * (D + 1) * tokens + B * c["Hq"] * D * (e + SIZE[c["out"]]) + 4.0 * sum((n + PAGE - 1) // PAGE for n in _lengths(c)),
                "flops": 4.0 * c["Hq"] * D * tokens}
    n = _tokens(c)
    new, row = 2.0 * B * Hkv * n, D + 1
    if c["kind"] == "write":
        past = 2.0 * B * Hkv * c["past"]
        return {"bytes": new * (D * e + row) + past * row + (new + past) * D * SIZE[c["out"]], "flops": 3.0 * (new + past) * D}
    rotated = float(B * n * D * (c["Hq"] + Hkv))
    table = 4.0 * n * D if c["kind"] == "rotate" else 4.0 * B * n * (D + len(c["sections"].split(",")))
    if c.get("pages") == "":
        return {"bytes": 2 * e * rotated + table, "flops": 3 * rotated}
    held = row if c.get("pages") != "bf16" else 2 * D
    return {"bytes": 2.0 * e * B * c["Hq"] * n * D + new * (D * e + held + 2 * D) + table, "flops": 3 * rotated + 3 * new * D}


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _row_values(x):
    """The rows that the 8-bit cache stands for, from the definition of the step: f64 [..., D] -> f64."""
    top = x.abs().amax(-1, keepdim=True)
    e = (torch.floor(torch.log2(torch.where(top > 0, top, 1.0) / 127.5)) + 1.0).clamp(min=-126.0)
    step = torch.exp2(e)
    return torch.round(x / step) * step


def _turned(x, cos, sin, interleaved):
    """The rotation whose products and sums are each rounded to 32 bits, as the operator is defined: complex numbers, f64."""
    def r(y):
        return y.float().double()

    n = x.shape[-1]
    first = torch.arange(n // 2, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else n // 2)
    re, im, c, s = x[..., first], x[..., second], cos.unsqueeze(1).double(), sin.unsqueeze(1).double()
    out = torch.empty_like(x)
    out[..., first], out[..., second] = r(r(re * c) - r(im * s)), r(r(im * c) + r(re * s))
    return out


def exact(case, seed):
    s, c = prepare(case, seed), case
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    if c["kind"] == "decode":
        g, got = c["Hq"] // Hkv, []
        for b in range(B):
            n = int(s["lens_host"][b])
            page = s["table_host"][b, :(n + PAGE - 1) // PAGE].cuda()
            k, v = (x[page].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :n] for x in (s["k"], s["v"]))
            ek, ev = (s["scales"][page][:, :, i].double().transpose(0, 1).reshape(Hkv, -1)[:, :n] - 127.0 for i in range(2))
            x = torch.einsum("hgd,hnd->hgn", s["q"][b, :, 0].double().view(Hkv, g, D), k * torch.exp2(ek)[..., None]) * s["scale"]
            weight = torch.softmax(x, -1)
            got.append(torch.einsum("hgn,hnd->hgd", weight, v * torch.exp2(ev)[..., None]).reshape(1, c["Hq"], 1, D))
        return torch.cat(got)
    if c["kind"] == "write":
        return tuple(_row_values(torch.cat([s[x + "0"], s[x]], 2).double()) for x in "kv")
    if c["kind"] == "rotate":
        cos, sin = s["cos"][None], s["sin"][None]
    else:
        axis, pair = torch.tensor(_axis_of_pair(c), device="cuda"), torch.arange(D // 2, device="cuda")
        at = s["positions"].long().permute(1, 2, 0)[..., axis]
        cos, sin = s["cos"][at, pair], s["sin"][at, pair]
    q, k = (_turned(s[x].double(), cos, sin, c["interleaved"]) for x in "qk")
    if c.get("pages") == "":
        return q, k
    if c.get("pages") == "bf16":
        return q, k, s["v"].double()
    return q, _row_values(k), _row_values(s["v"].double())
