"""The operators on 4-bit weights and 4-bit key/value caches, as cases to measure.

The 4-bit format: values of 1 sign, 2 exponent and 1 mantissa bits (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives), two to a byte with the lower index in the low half, in blocks of 32 along a row; each block has one
scale byte s, a factor of 2^(s - 127). A row whose length is no multiple of 32 ends in a block padded with zeros.

- product: y = x W + b with W in 4 bits, one row (a decode step) to thousands (a prompt);
- append: the key and value columns of packed QKV rows rounded into a 4-bit cache at each sequence's own
  position, and read back;
- attention: queries against a 4-bit cache with grouped heads and sequences of their own lengths, one new token a
  sequence (a decode step) or a chunk of a prompt, causal.

Sizes: the widths of the model configurations the benchmark and the tests use (512 and 768, 16 codebooks of 1024
classes, head dims 32 and 64, caches of 1408 positions), larger ones of serving in general, and ragged ones.
"""
import ctypes
import math
import random

import torch

own = False  # False: the plain forms; True: the framework's operators

BLOCK = 32


# ---- the cases -----------------------------------------------------------------------------------


def listed():
    return [
        # One token's QKV projection of the 111.5M-model: the latency of a decode step's products.
        dict(name="product_1x768x2304", kind="product", rows=1, inner=768, cols=2304, bf16=False),
        # One token's 16-codebook head: the largest weight of that model for a single row.
        dict(name="product_1x768x16384", kind="product", rows=1, inner=768, cols=16384, bf16=False),
        # Sixteen sequences decoded together through a wide layer.
        dict(name="product_16x4096x14336", kind="product", rows=16, inner=4096, cols=14336, bf16=False),
        # One token through a large layer's 125 MB of weights: the rate at which weights are read.
        dict(name="product_1x8192x28672", kind="product", rows=1, inner=8192, cols=28672, bf16=False),
        # A prompt's tokens through a square layer: matrix-bound.
        dict(name="product_2048x4096x4096", kind="product", rows=2048, inner=4096, cols=4096, bf16=False),
        # A ragged prompt with inputs rounded to bf16, odd widths (rows of no 16-byte alignment).
        dict(name="product_bf16_777x1001x1537", kind="product", rows=777, inner=1001, cols=1537, bf16=True),
        # Sixteen sequences' new tokens into their caches, each at its own position.
        dict(name="append_16x1", kind="append", batch=16, time=1, kv_heads=8, head_dim=128, capacity=8192, ragged=3),
        # A prompt's chunk into the medium model's cache (head dim 64).
        dict(name="append_4x2000", kind="append", batch=4, time=2000, kv_heads=8, head_dim=64, capacity=4096, ragged=5),
        # The 111.5M-model's decode step: one query a head against 701 positions.
        dict(name="attention_1x12_701", kind="attention", batch=1, heads=12, kv_heads=12, head_dim=64, queries=1,
             capacity=1408, longest=701, ragged=0),
        # Sixteen sequences of different lengths decoded together, four query heads to a key/value head.
        dict(name="attention_16x32_ragged", kind="attention", batch=16, heads=32, kv_heads=8, head_dim=128, queries=1,
             capacity=8192, longest=8192, ragged=7),
        # One long sequence, eight query heads to a key/value head.
        dict(name="attention_1x64_131071", kind="attention", batch=1, heads=64, kv_heads=8, head_dim=128, queries=1,
             capacity=131072, longest=131071, ragged=0),
        # Two prompts' 1000-token chunks against what is cached of them.
        dict(name="attention_2x16_chunk", kind="attention", batch=2, heads=16, kv_heads=4, head_dim=128, queries=1000,
             capacity=6144, longest=6001, ragged=9),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A layer width: a multiple of 128, a multiple of 32, or any number."""
    n = _log_int(rng, low, high)
    step = rng.choice([128, 128, 32, 1])
    return max(step, n // step * step)


MAX_FLOPS = 6.8e10   # of the largest listed product
MAX_BYTES = 1.2e8    # of the largest listed product's weights; of the longest listed cache
MAX_APPEND = 7e7     # of the largest listed append
MAX_HELD = 1.35e8    # of the longest listed cache's keys


def _large(case):
    """Whether an attention case passes the largest listed ones, in what it moves, computes or holds."""
    queries, values = case["heads"] * case["queries"], case["kv_heads"] * case["head_dim"]
    return (work(case)["bytes"] > MAX_BYTES or work(case)["flops"] > MAX_FLOPS
            or case["batch"] * case["capacity"] * max(values, queries) > MAX_HELD)


def draw(rng):
    kind = rng.choice(["product", "product", "product", "append", "attention", "attention", "attention"])
    if kind == "product":
        few = rng.random() < 0.6
        case = dict(kind=kind, rows=_log_int(rng, 1, 32) if few else _log_int(rng, 33, 3000),
                    inner=_width(rng, 64, 8192), cols=_width(rng, 64, 28672), bf16=rng.random() < 0.25)
        while work(case)["flops"] > MAX_FLOPS or work(case)["bytes"] > MAX_BYTES:
            case["cols"] = max(16, case["cols"] * 2 // 3)
            case["rows"] = max(1, case["rows"] * 3 // 4) if not few else case["rows"]
        return case
    head_dim = rng.choice([32, 64, 64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    if kind == "append":
        capacity = _log_int(rng, 64, 8192)
        case = dict(kind=kind, batch=_log_int(rng, 1, 16), time=rng.choice([1, _log_int(rng, 1, min(capacity, 2000))]),
                    kv_heads=min(kv_heads, 8), head_dim=head_dim, capacity=capacity, ragged=rng.randint(1, 10 ** 6))
        while work(case)["bytes"] > MAX_APPEND:
            case["time"] = case["time"] * 2 // 3
        return case
    queries = 1 if rng.random() < 0.6 else _log_int(rng, 2, 1000)
    longest = _log_int(rng, max(16, queries), 65536 if queries == 1 else 4096)
    case = dict(kind=kind, batch=_log_int(rng, 1, 16 if queries == 1 else 3), heads=kv_heads * rng.choice([1, 1, 2, 4, 8]),
                kv_heads=kv_heads, head_dim=head_dim, queries=queries, capacity=longest + rng.randint(0, 512),
                longest=longest, ragged=rng.randint(0, 10 ** 6))
    while _large(case) and case["batch"] > 1:
        case["batch"] -= 1
    if _large(case):
        case["heads"], case["kv_heads"] = case["heads"] // case["kv_heads"], 1
    return case


def _lengths(case):
    """The positions each sequence holds, the new tokens among them: all `longest`, or (ragged) from the number of
    new tokens to `longest`, spread over the logarithm; of a ragged decode batch the second place is free (0)."""
    if not case["ragged"]:
        return [case["longest"]] * case["batch"]
    rng = random.Random(case["ragged"])
    got = [_log_int(rng, case["queries"], case["longest"]) for _ in range(case["batch"])]
    got[0] = case["longest"]
    if case["queries"] == 1 and case["batch"] > 1:
        got[1] = 0
    return got


def _positions(case):
    """Where each sequence's new tokens go: any place that holds them all."""
    rng = random.Random(case["ragged"])
    return [rng.randint(0, case["capacity"] - case["time"]) for _ in range(case["batch"])]


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    """Bytes: inputs read once, results written once. Flops: multiply-adds over what the mask shows."""
    if case["kind"] == "product":
        m, k, n = case["rows"], case["inner"], case["cols"]
        return dict(bytes=4 * (m * k + n + m * n) + 17 * n * -(-k // BLOCK), flops=2 * m * k * n)
    if case["kind"] == "append":
        values = 2 * case["batch"] * case["time"] * case["kv_heads"] * case["head_dim"]
        return dict(bytes=values * 4 * 2 + values // BLOCK * 17, flops=4 * values)
    t, h = case["queries"], case["head_dim"]
    held = sum(_lengths(case))
    pairs = sum(t * n - t * (t - 1) // 2 for n in _lengths(case) if n >= t)
    return dict(bytes=2 * held * case["kv_heads"] * h // BLOCK * 17 + 8 * case["batch"] * t * case["heads"] * h,
                flops=4 * pairs * case["heads"] * h)


# ---- the format in plain operations --------------------------------------------------------------------


def _power(e):
    """2^e for whole e in -127 .. 127, from its bits."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _pack(v):
    """[..., n] floats -> codes [..., ceil(n / 32) * 16] and scales [..., ceil(n / 32)], uint8."""
    v = torch.nn.functional.pad(v, (0, -v.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    mantissa, exponent = torch.frexp(v.abs().amax(-1))  # the largest = mantissa 2^exponent, mantissa in [0.5, 1)
    e = exponent.int() - 3 + (mantissa >= 0.875).int()   # the smallest power of two of which it is under 7
    e = torch.where(mantissa == 0, torch.full_like(e, -127), e.clamp(min=-127))
    a = v.abs() * _power(-e)[..., None]
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5).int() + 8 * torch.signbit(v).int())
    code = code.flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), (e + 127).to(torch.uint8)


def _unpack(codes, scales):
    """The values the codes stand for, fp32, [..., blocks * 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    values = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2)
    return (values.unflatten(-1, (-1, BLOCK)) * _power(scales.int() - 127)[..., None]).flatten(-2)


# ---- inputs --------------------------------------------------------------------------------------


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=generator, device="cuda", dtype=torch.float32).mul_(std)

    def empty(*shape):
        return torch.empty(*shape, device="cuda", dtype=torch.float32)

    state = dict(case=case)
    if case["kind"] == "product":  # N(0, 1) activations, N(0, 0.02) weights, as the models start with
        m, k, n = case["rows"], case["inner"], case["cols"]
        state.update(x=normal(m, k), bias=normal(n, std=0.02), y=empty(m, n))
        state["codes"], state["scales"] = _pack(normal(n, k, std=0.02))
    elif case["kind"] == "append":
        b, t, n, h, c = (case[name] for name in ("batch", "time", "kv_heads", "head_dim", "capacity"))
        state.update(qkv=normal(b * t, 3 * n * h), positions=torch.tensor(_positions(case), device="cuda").int(),
                     k=empty(b, n, t, h), v=empty(b, n, t, h))
        for name in ("k", "v"):
            state[name + "_codes"] = torch.zeros(b, n, c, h // 2, device="cuda", dtype=torch.uint8)
            state[name + "_scales"] = torch.zeros(b, n, c, h // BLOCK, device="cuda", dtype=torch.uint8)
    else:
        b, n, kv, t, h, c = (case[name] for name in ("batch", "heads", "kv_heads", "queries", "head_dim", "capacity"))
        lengths = torch.tensor(_lengths(case), device="cuda").int()
        state.update(q=normal(b, t, n, h), out=empty(b, t, n, h), lengths=lengths)
        held = torch.arange(c, device="cuda") < lengths[:, None]
        for name in ("k", "v"):  # positions past a sequence's length were never written
            codes, scales = _pack(normal(b, kv, c, h) * held[:, None, :, None])
            state[name + "_codes"], state[name + "_scales"] = codes, scales
    torch.cuda.synchronize()  # the library runs on a stream of its own
    return state


# ---- one pass ------------------------------------------------------------------------------------


def _product(s):
    x = s["x"].bfloat16().float() if s["case"]["bf16"] else s["x"]
    w = _unpack(s["codes"], s["scales"])[:, :s["case"]["inner"]]
    return x @ w.t() + s["bias"]


def _append(s):
    b, t, n, h = (s["case"][name] for name in ("batch", "time", "kv_heads", "head_dim"))
    at = s["positions"].long()[:, None] + torch.arange(t, device="cuda")
    sequence = torch.arange(b, device="cuda")[:, None]
    columns = s["qkv"].view(b, t, 3, n, h)
    got = {}
    for part, name in ((1, "k"), (2, "v")):
        codes, scales = _pack(columns[:, :, part])
        s[name + "_codes"][sequence, :, at] = codes
        s[name + "_scales"][sequence, :, at] = scales
        got[name] = _unpack(s[name + "_codes"][sequence, :, at], s[name + "_scales"][sequence, :, at]).transpose(1, 2)
    return got


def _attention(s):
    b, n, kv, t, h, c = (s["case"][name] for name in ("batch", "heads", "kv_heads", "queries", "head_dim", "capacity"))
    k, v = _unpack(s["k_codes"], s["k_scales"]), _unpack(s["v_codes"], s["v_scales"])
    q = s["q"].view(b, t, kv, n // kv, h).transpose(1, 2).reshape(b, kv, t * (n // kv), h)
    scores = q @ k.transpose(2, 3) * h ** -0.5
    last = s["lengths"][:, None] - t + torch.arange(t, device="cuda")  # the last key each query sees
    visible = torch.arange(c, device="cuda") <= last[:, :, None]
    visible = visible.repeat_interleave(n // kv, 1)[:, None]
    largest = scores.masked_fill(~visible, -math.inf).amax(-1, keepdim=True)
    p = torch.exp(scores - largest).masked_fill(~visible, 0.0)
    total = p.sum(-1, keepdim=True)
    out = p @ v / torch.where(total > 0, total, torch.ones_like(total))  # a query that sees nothing gives zeros
    return out.view(b, kv, t, n // kv, h).transpose(1, 2).reshape(b, t, n, h)


_GPU = None


def _calls(s):
    """The library's calls for this state, arguments built once, as a compiled program holds them."""
    global _GPU
    from staleynet_amd import gemm

    if _GPU is None:
        _GPU = gemm.Gpu(0)
    case, library, keep = s["case"], gemm.library(), []

    def call(name, *args):
        flat = [_GPU._ctx]
        for a in args:
            if isinstance(a, torch.Tensor):
                flat += [ctypes.c_void_p(a.data_ptr()), ctypes.c_size_t(a.numel())]
            elif isinstance(a, ctypes.Structure):
                keep.append(a)
                flat.append(ctypes.byref(a))
            else:
                flat.append(a)
        return getattr(library, name), tuple(flat), keep

    if case["kind"] == "product":
        precision = gemm.Precision.Bf16 if case["bf16"] else gemm.Precision.F32
        spec = gemm.MatmulSpec.new(case["rows"], case["cols"], case["inner"]).right_transposed()
        return [call("sn_matmul_fp4", spec.with_precision(precision).to_c(), s["x"], s["codes"], s["scales"],
                     s["bias"], s["y"])], s["y"]
    buffers = [s[name + part] for name in ("k", "v") for part in ("_codes", "_scales")]
    cache = gemm.CFp4CacheShape(case["batch"], case["kv_heads"], case["capacity"], case["head_dim"])
    if case["kind"] == "append":
        width = 3 * case["kv_heads"] * case["head_dim"]
        rows = gemm.CFp4CacheRows(case["time"], 0, width, width // 3, 2 * width // 3)
        return [call("sn_fp4_cache_append", cache, rows, s["qkv"], s["positions"], *buffers),
                call("sn_fp4_cache_read", cache, rows, *buffers, s["positions"], s["k"], s["v"])], \
            dict(k=s["k"], v=s["v"])
    t, n, h = case["queries"], case["heads"], case["head_dim"]
    shape = gemm.CFp4AttentionShape(n, t, 0, t * n * h, h, n * h, t * n * h, h, n * h, h ** -0.5)
    return [call("sn_fp4_attention", cache, shape, s["q"], *buffers, s["lengths"], s["out"])], s["out"]


def run(state):
    if own:
        if "calls" not in state:
            state["calls"] = _calls(state)
        calls, outputs = state["calls"]
        for function, args, _ in calls:
            status = function(*args)
            if status != 0:
                raise RuntimeError("status %d" % status)
        return outputs
    return dict(product=_product, append=_append, attention=_attention)[state["case"]["kind"]](state)


# ---- the same in 64 bits -----------------------------------------------------------------------------


def _values64(codes, scales):
    """The codes' values from the format's definition: (-1)^sign 2^(exponent - 1) (1 + mantissa / 2), or mantissa / 2."""
    code = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    sign, exponent, mantissa = 1.0 - 2.0 * (code // 8), code // 2 % 4, (code % 2).double()
    magnitude = torch.where(exponent == 0, mantissa / 2, torch.exp2(exponent.double() - 1) * (1 + mantissa / 2))
    scale = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)
    return sign * magnitude * scale


def _rounded64(v):
    """Values as a 4-bit cache holds them: multiples of 0.5, 1 or 2 of the block's power of two, ties to even."""
    v = v.double().unflatten(-1, (-1, BLOCK))
    largest = v.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(largest)) - 2)
    unit = torch.where(largest / unit >= 7, 2 * unit, unit)
    a = v / unit
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0)).double()
    return ((torch.round(a / step) * step).clamp(-6, 6) * unit).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "product":
        x = (s["x"].bfloat16() if case["bf16"] else s["x"]).double()
        return x @ _values64(s["codes"], s["scales"])[:, :case["inner"]].T.contiguous() + s["bias"].double()
    if case["kind"] == "append":
        b, t, n, h = (case[name] for name in ("batch", "time", "kv_heads", "head_dim"))
        k, v = (_rounded64(part.reshape(b, t, n, h)).permute(0, 2, 1, 3) for part in s["qkv"].chunk(3, 1)[1:])
        return dict(k=k, v=v)
    t, h, group = case["queries"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for b, length in enumerate(_lengths(case)):
        if length == 0:
            continue
        hidden = torch.ones(t, length, device="cuda", dtype=torch.bool).triu_(length - t + 1)
        for head in range(case["kv_heads"]):
            k, v = (_values64(s[name + "_codes"][b, head, :length], s[name + "_scales"][b, head, :length])
                    for name in ("k", "v"))
            for query in range(head * group, (head + 1) * group):
                weights = (s["q"][b, :, query].double() @ k.T.contiguous() / math.sqrt(h)).masked_fill_(hidden, -math.inf)
                out[b, :, query] = torch.softmax(weights, -1) @ v
    return out
