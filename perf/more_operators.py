"""The operators from the residual stream to answered tokens, as cases to measure.

The 8-bit format: e4m3 values (1 sign, 4 exponent, 3 mantissa bits, largest 448) in blocks of 128 along a row; each
block has one scale byte s, a factor of 2^(s - 127), the smallest power of two of which the block's largest magnitude
is at most 464 (what rounds to 448). A row ends in a block padded with zeros, its scale bytes are padded to fours.

- norm: the residual stream's addition s = x + r and its root-mean-square norm y = w s / sqrt(mean(s^2) + eps), y
  rounded to the 8-bit format (and read back), or in 32 bits; its gradients;
- quantize: rows or a weight's columns rounded to the 8-bit format, and read back;
- product: y = x W + b with both operands in that format, one row (a decode step) to thousands (a prompt);
- logprobs: per token and head the log probability of a given class, the entropy and the likeliest classes, from the
  rows of logits that such a product leaves; their gradient.

Sizes: the widths of the model configurations the benchmark and the tests use (512 and 768, 16 codebooks of 1024
classes), larger ones of serving in general, and ragged ones.
"""
import ctypes
import math
import random

import torch

own = False  # False: the plain forms; True: the framework's operators

BLOCK = 128
LARGEST_SCALE = 246
EMPTY = -1  # a place without a token, 0xFFFFFFFF
EPSILON = 9.999999747378752e-06  # 1e-5 in 32 bits


# ---- the cases -----------------------------------------------------------------------------------


def listed():
    return [
        # One token's residual addition and norm before the 111.5M model's QKV: the latency of a decode step's norms.
        dict(name="norm_1x768", kind="norm", rows=1, width=768, eight=True),
        # A prompt's tokens through a wide layer's norm: memory-bound.
        dict(name="norm_8192x4096", kind="norm", rows=8192, width=4096, eight=True),
        # The norm's gradients over a training batch of the 111.5M model.
        dict(name="norm_backward_8192x768", kind="norm_backward", rows=8192, width=768),
        # A ragged batch of activations to 8 bits before a layer, rows of no 16-byte alignment.
        dict(name="quantize_rows_1999x4001", kind="quantize", rows=1999, inner=4001, transposed=False),
        # A wide layer's weight to 8 bits, its columns as rows: what a training step does with each weight.
        dict(name="quantize_weight_14336x4096", kind="quantize", rows=14336, inner=4096, transposed=True),
        # One token's QKV projection of the 111.5M model: the latency of a decode step's products.
        dict(name="product_1x768x2304", kind="product", rows=1, inner=768, cols=2304),
        # Sixteen sequences decoded together through a wide layer: the rate at which weights are read.
        dict(name="product_16x4096x14336", kind="product", rows=16, inner=4096, cols=14336),
        # A ragged prompt through the same layer: matrix-bound.
        dict(name="product_6001x4096x14336", kind="product", rows=6001, inner=4096, cols=14336),
        # One decode step's 16 codebooks of 1024 classes: the sampled codes' log probabilities and five alternatives.
        dict(name="logprobs_1x16x1024", kind="logprobs", rows=1, heads=16, classes=1024, offset=0, top=5, scale=1.0),
        # A batch of answers scored over a large vocabulary at a temperature, twenty alternatives each.
        dict(name="logprobs_128x131072", kind="logprobs", rows=128, heads=1, classes=131072, offset=0, top=20, scale=0.8),
        # The gradient of sampled codes' log probabilities and of the entropy, a training batch of the model.
        dict(name="logprobs_backward_4096x16x1024", kind="logprobs_backward", rows=4096, heads=16, classes=1024, offset=0,
             scale=1.0),
        # The same over a ragged vocabulary whose rows have no 16-byte alignment.
        dict(name="logprobs_backward_333x50001", kind="logprobs_backward", rows=333, heads=1, classes=50001, offset=3,
             scale=0.8),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A layer width: a multiple of 128, a multiple of 16, or any number."""
    n = _log_int(rng, low, high)
    step = rng.choice([128, 128, 16, 1])
    return max(step, n // step * step)


MAX_BYTES = dict(norm=4.0e8, norm_backward=1.2e8, quantize=4.5e8, product=4.5e8, logprobs=6.5e7,
                 logprobs_backward=5.2e8)  # of the largest listed case of each kind, or under it
MAX_FLOPS = 7.0e11


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_backward", "quantize", "product", "product", "product", "logprobs",
                       "logprobs", "logprobs_backward"])
    if kind in ("norm", "norm_backward"):
        case = dict(kind=kind, rows=_log_int(rng, 1, 16384), width=_width(rng, 64, 16384))
        if kind == "norm":
            case["eight"] = rng.random() < 0.7
        shrink = "rows"
    elif kind == "quantize":
        case = dict(kind=kind, rows=_log_int(rng, 1, 16384), inner=_width(rng, 64, 16384), transposed=rng.random() < 0.5)
        shrink = "rows"
    elif kind == "product":
        few = rng.random() < 0.5
        case = dict(kind=kind, rows=_log_int(rng, 1, 64) if few else _log_int(rng, 65, 8192),
                    inner=_width(rng, 64, 16384), cols=_width(rng, 64, 28672))
        shrink = "cols"
    else:
        books = rng.random() < 0.5  # codebooks of one model, or one vocabulary
        case = dict(kind=kind, rows=_log_int(rng, 1, 4096), heads=rng.randint(2, 16) if books else 1,
                    classes=_log_int(rng, 60, 2100) if books else _log_int(rng, 1000, 262144),
                    offset=rng.choice([0, 0, 4, rng.randint(1, 999)]))
        if rng.random() < 0.5:
            case["classes"] = max(64, case["classes"] // 64 * 64)
        if kind == "logprobs":
            case["top"] = rng.choice([0, 1, 5, 20, rng.randint(2, 32)])
        case["scale"] = rng.choice([1.0, 1.0, 0.7, 1.25])
        shrink = "rows"
    while work(case)["bytes"] > MAX_BYTES[kind] or work(case)["flops"] > MAX_FLOPS:
        case[shrink] = max(1, case[shrink] * 2 // 3)
    return case


# ---- what a pass cannot do without ------------------------------------------------------------------


def _blocks(inner):
    return -(-inner // BLOCK)


def _row_bytes(inner):
    """Bytes of one row of the 8-bit format: its codes and its scale bytes."""
    return _blocks(inner) * BLOCK + -(-_blocks(inner) // 4) * 4


def work(case):
    """Bytes: inputs read once, results written once. Flops: multiplies, additions and exponentials of the formulas."""
    if case["kind"] == "norm":  # x, r and w read; s and the 8-bit rows (and their values) or y written
        n, w = case["rows"], case["width"]
        return dict(bytes=4 * (4 * n * w + w) + (n * _row_bytes(w) if case["eight"] else 0), flops=6 * n * w)
    if case["kind"] == "norm_backward":  # s, dy and the gradient that meets s read, ds and dw written
        n, w = case["rows"], case["width"]
        return dict(bytes=4 * (4 * n * w + n + 2 * w), flops=10 * n * w)
    if case["kind"] == "quantize":
        n, k = case["rows"], case["inner"]
        return dict(bytes=8 * n * k + n * _row_bytes(k), flops=3 * n * k)
    if case["kind"] == "product":
        m, k, n = case["rows"], case["inner"], case["cols"]
        return dict(bytes=(m + n) * _row_bytes(k) + 4 * n + 4 * m * n, flops=2 * m * k * n)
    n = case["rows"] * case["heads"]
    if case["kind"] == "logprobs":
        return dict(bytes=4 * n * case["classes"] + 4 * n * (1 + 1 + 1 + 2 + 2 * case["top"]), flops=6 * n * case["classes"])
    return dict(bytes=8 * n * case["classes"] + 4 * n * (1 + 2 + 1 + 2), flops=10 * n * case["classes"])


# ---- the format in plain operations --------------------------------------------------------------------


def _power(e):
    """2^e for whole e in -127 .. 127, from its bits."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _pack(v):
    """[..., n] floats -> codes [..., blocks * 128] and scales [..., blocks rounded up to fours], uint8."""
    v = torch.nn.functional.pad(v, (0, -v.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    mantissa, exponent = torch.frexp(v.abs().amax(-1))       # the largest = mantissa 2^exponent, mantissa in [0.5, 1)
    e = exponent.int() - 9 + (mantissa > 0.90625).int()      # the smallest power of two of which it is at most 464
    e = torch.where(mantissa == 0, torch.full_like(e, -127), e.clamp(min=-127, max=LARGEST_SCALE - 127))
    a = (v.abs() * _power(-e)[..., None]).clamp(max=448)
    at = torch.frexp(a.clamp(min=2.0 ** -6))[1].int()        # the binade; values under 2^-6 are in the smallest's steps
    units = torch.round(a / _power(at - 4)).int()            # of 3 mantissa bits, ties to even; 8 .. 16, under 2^-6 0 .. 8
    code = (at + 5) * 8 + units + 128 * torch.signbit(v).int()  # 16 units are the next exponent's 8
    scales = (e + 127).to(torch.uint8)
    return code.to(torch.uint8).flatten(-2), torch.nn.functional.pad(scales, (0, -scales.shape[-1] % 4))


def _unpack(codes, scales, inner):
    """The values the codes stand for, fp32, [..., inner]."""
    code = torch.arange(256, device="cuda")
    exponent, mantissa = code // 8 % 16, (code % 8).float()
    table = torch.where(exponent == 0, mantissa, mantissa + 8) * _power((exponent.clamp(min=1) - 10).int())
    table = torch.where(code >= 128, -table, table)
    values = table[codes.int()].unflatten(-1, (-1, BLOCK))
    return (values * _power(scales[..., :values.shape[-2]].int() - 127)[..., None]).flatten(-2)[..., :inner]


# ---- inputs --------------------------------------------------------------------------------------


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=generator, device="cuda", dtype=torch.float32).mul_(std).add_(mean)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    def pattern(rows, inner):
        return dict(codes=empty(rows, _blocks(inner) * BLOCK, dtype=torch.uint8),
                    scales=empty(rows, -(-_blocks(inner) // 4) * 4, dtype=torch.uint8))

    state = dict(case=case)
    kind = case["kind"]
    if kind == "norm":  # a residual stream of some depth, a layer's output that joins it, weights about one
        n, w = case["rows"], case["width"]
        state.update(x=normal(n, w), residual=normal(n, w, std=3.0), weight=normal(w, std=0.1, mean=1.0), sum=empty(n, w),
                     y=empty(n, w))
        if case["eight"]:
            state.update(pattern(n, w))
    elif kind == "norm_backward":
        n, w = case["rows"], case["width"]
        state.update(sum=normal(n, w, std=3.0), weight=normal(w, std=0.1, mean=1.0), d_out=normal(n, w, std=1e-3),
                     d_sum=normal(n, w, std=1e-3), d_x=empty(n, w), d_weight=empty(w))
        state["inverse"] = ((state["sum"].double() ** 2).mean(-1) + EPSILON).rsqrt().float()  # the forward leaves it
    elif kind == "quantize":
        n, k = case["rows"], case["inner"]
        shape = (k, n) if case["transposed"] else (n, k)
        state.update(pattern(n, k), source=normal(*shape, std=0.02 if case["transposed"] else 1.0), back=empty(*shape))
    elif kind == "product":  # N(0, 1) activations, N(0, 0.02) weights, as the models start with
        m, k, n = case["rows"], case["inner"], case["cols"]
        state.update(bias=normal(n, std=0.02), y=empty(m, n))
        state["left_codes"], state["left_scales"] = _pack(normal(m, k))
        state["right_codes"], state["right_scales"] = _pack(normal(n, k, std=0.02))
    else:
        n, heads, classes = case["rows"], case["heads"], case["classes"]
        cols = case["offset"] + heads * classes
        logits = normal(n, cols, std=3.0)
        # Classes that may not be answered (one in 64) are at minus infinity, the answered ones are not of them; some
        # places have no token.
        masked = torch.rand(cols, generator=generator, device="cuda") < 1 / 64
        logits[:, masked] = -math.inf
        tokens = torch.randint(0, classes, (n, heads), generator=generator, device="cuda")
        columns = case["offset"] + classes * torch.arange(heads, device="cuda") + tokens
        logits.scatter_(1, columns, normal(n, heads, std=3.0))
        tokens = tokens.int()
        tokens[torch.rand(n, heads, generator=generator, device="cuda") < 1 / 16] = EMPTY
        state.update(logits=logits, tokens=tokens)
        if kind == "logprobs":
            top = case["top"]
            state.update(logprobs=empty(n, heads), entropies=empty(n, heads), stats=empty(n, heads, 2))
            if top:
                state.update(top_tokens=empty(n, heads, top, dtype=torch.int32), top_logprobs=empty(n, heads, top))
        else:  # what the forward leaves, and gradients of a loss of both
            z = logits[:, case["offset"]:].view(n, heads, classes)
            largest = z.amax(-1)
            p = torch.exp((z - largest[..., None]) * case["scale"])
            total = p.sum(-1, dtype=torch.float64)
            weighted = torch.where(p > 0, p * (z - largest[..., None]), torch.zeros_like(p)).sum(-1, dtype=torch.float64)
            state.update(stats=torch.stack([largest, torch.log(total).float()], -1).contiguous(),
                         entropies=(torch.log(total) - case["scale"] * weighted / total).float(),
                         d_logprobs=normal(n, heads), d_entropies=normal(n, heads, std=0.1), grad=torch.zeros_like(logits))
    torch.cuda.synchronize()  # the library runs on a stream of its own
    return state


# ---- one pass ------------------------------------------------------------------------------------


def _norm(s):
    total = s["x"] + s["residual"]
    wide = total.double() if s["case"]["eight"] else total  # codes next to a border
    y = (wide * torch.rsqrt((wide * wide).mean(-1, keepdim=True) + EPSILON) * s["weight"]).float()
    if s["case"]["eight"]:
        y = _unpack(*_pack(y), s["case"]["width"])
    return dict(sum=total, y=y)


def _norm_backward(s):
    inverse = s["inverse"][:, None]
    normed = s["sum"] * inverse
    g = s["d_out"] * s["weight"]
    d_x = s["d_sum"] + inverse * (g - normed * (g * normed).mean(-1, keepdim=True))
    return dict(d_x=d_x, d_weight=(s["d_out"] * normed).sum(0))


def _quantize(s):
    source = s["source"].t() if s["case"]["transposed"] else s["source"]
    back = _unpack(*_pack(source), s["case"]["inner"])
    return back.t().contiguous() if s["case"]["transposed"] else back


def _product(s):
    x = _unpack(s["left_codes"], s["left_scales"], s["case"]["inner"])
    w = _unpack(s["right_codes"], s["right_scales"], s["case"]["inner"])
    return x @ w.t() + s["bias"]


def _heads(s):
    case = s["case"]
    return s["logits"][:, case["offset"]:].reshape(case["rows"], case["heads"], case["classes"])


def _logprobs(s):
    scale, top, tokens = s["case"]["scale"], s["case"]["top"], s["tokens"].long()
    z = _heads(s)
    largest = z.amax(-1, keepdim=True)
    shifted = (z - largest) * scale
    p = torch.exp(shifted)
    total = p.sum(-1)
    log_total = torch.log(total)
    got = shifted.gather(-1, tokens.clamp(min=0)[..., None])[..., 0] - log_total
    weighted = torch.where(p > 0, p * shifted, torch.zeros_like(p)).sum(-1)
    out = dict(logprobs=torch.where(tokens < 0, torch.zeros_like(got), got), entropies=log_total - weighted / total,
               stats=torch.stack([largest[..., 0], log_total], -1))
    if top:
        order = torch.sort(z, dim=-1, descending=True, stable=True)[1][..., :top]  # ties to the lower class
        out.update(top_tokens=order.int(), top_logprobs=shifted.gather(-1, order) - log_total[..., None])
    return out


def _logprobs_backward(s):
    case, tokens = s["case"], s["tokens"].long()
    log_p = (_heads(s) - s["stats"][..., :1]) * case["scale"] - s["stats"][..., 1:]
    p = torch.exp(log_p)
    d_logprobs = torch.where(tokens < 0, torch.zeros_like(s["d_logprobs"]), s["d_logprobs"])[..., None]
    grad = -p * d_logprobs - torch.where(p > 0, s["d_entropies"][..., None] * p * (log_p + s["entropies"][..., None]),
                                         torch.zeros_like(p))
    grad.scatter_add_(-1, tokens.clamp(min=0)[..., None], d_logprobs)
    out = torch.zeros_like(s["logits"])
    out[:, case["offset"]:] = (grad * case["scale"]).flatten(1)
    return out


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
            if isinstance(a, str):  # a buffer of the state, or none
                t = s.get(a)
                flat += [None, ctypes.c_size_t(0)] if t is None else \
                    [ctypes.c_void_p(t.data_ptr()), ctypes.c_size_t(t.numel())]
            elif isinstance(a, ctypes.Structure):
                keep.append(a)
                flat.append(ctypes.byref(a))
            else:
                flat.append(a)
        return getattr(library, name), tuple(flat), keep

    kind = case["kind"]
    if kind == "norm":
        shape = gemm.CRmsNormShape(case["rows"], case["width"], EPSILON)
        outputs = dict(sum=s["sum"], y=s["y"])
        if not case["eight"]:
            return [call("sn_rms_norm", shape, "x", "residual", "weight", "sum", "y", "none")], outputs
        return [call("sn_rms_norm_fp8", shape, "x", "residual", "weight", "sum", "codes", "scales"),
                call("sn_dequantize_fp8", case["rows"], case["width"], int(gemm.Storage.RowMajor), "codes", "scales",
                     "y")], outputs
    if kind == "norm_backward":
        shape = gemm.CRmsNormShape(case["rows"], case["width"], EPSILON)
        zero = gemm.library().sn_fill_zero, (_GPU._ctx, ctypes.c_void_p(s["d_weight"].data_ptr()),
                                             ctypes.c_size_t(case["width"])), keep  # the gradient is added to
        return [zero, call("sn_rms_norm_backward", shape, "sum", "inverse", "weight", "d_out", "d_sum", "d_x", "d_weight")], \
            dict(d_x=s["d_x"], d_weight=s["d_weight"])
    if kind == "quantize":
        storage = int(gemm.Storage.Transposed if case["transposed"] else gemm.Storage.RowMajor)
        return [call("sn_quantize_fp8", case["rows"], case["inner"], storage, "source", "codes", "scales"),
                call("sn_dequantize_fp8", case["rows"], case["inner"], storage, "codes", "scales", "back")], s["back"]
    if kind == "product":
        spec = gemm.MatmulSpec.new(case["rows"], case["cols"], case["inner"]).right_transposed()
        return [call("sn_matmul_fp8", spec.to_c(), "left_codes", "left_scales", "right_codes", "right_scales", "bias",
                     "y")], s["y"]
    shape = gemm.CLogprobShape(case["rows"], case["offset"] + case["heads"] * case["classes"], case["offset"],
                               case["classes"], case["heads"], case["heads"], 0, case.get("top", 0), case["scale"])
    if kind == "logprobs":
        names = ("logprobs", "entropies", "stats", "top_tokens", "top_logprobs")
        return [call("sn_token_logprobs", shape, "logits", "tokens", *names)], \
            {name: s[name] for name in names if name in s}
    return [call("sn_token_logprobs_backward", shape, "logits", "tokens", "stats", "entropies", "d_logprobs",
                 "d_entropies", "grad")], s["grad"]


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
    return dict(norm=_norm, norm_backward=_norm_backward, quantize=_quantize, product=_product, logprobs=_logprobs,
                logprobs_backward=_logprobs_backward)[state["case"]["kind"]](state)


# ---- the same in 64 bits -----------------------------------------------------------------------------


def _values64(codes, scales, inner):
    """The codes' values from the format's definition: (-1)^sign 2^(exponent - 7) (1 + mantissa / 8), or 2^-6 mantissa / 8."""
    code = codes.long()
    sign, exponent, mantissa = 1.0 - 2.0 * (code // 128), code // 8 % 16, (code % 8).double()
    magnitude = torch.where(exponent == 0, mantissa / 512, torch.exp2(exponent.double() - 7) * (1 + mantissa / 8))
    scale = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]
    return (sign * magnitude * scale)[..., :inner]


def _rounded64(v):
    """Values as the format holds them: multiples of the step of each binade of the block's power of two, ties to even."""
    n = v.shape[-1]
    v = torch.nn.functional.pad(v.double(), (0, -n % BLOCK)).unflatten(-1, (-1, BLOCK))
    largest = v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -160)
    unit = torch.exp2(torch.ceil(torch.log2(largest / 464)).clamp(-127, LARGEST_SCALE - 127))
    a = v / unit
    step = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6))) - 3)
    return ((torch.round(a / step) * step).clamp(-448, 448) * unit).flatten(-2)[..., :n]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        total = s["x"] + s["residual"]  # rounded once, as the stream is kept in 32 bits
        wide = total.double()
        y = wide / torch.sqrt(wide.square().mean(-1, keepdim=True) + EPSILON) * s["weight"].double()
        return dict(sum=total, y=_rounded64(y.float()) if case["eight"] else y)
    if kind == "norm_backward":
        x, inverse, w, g = (s[name].double() for name in ("sum", "inverse", "weight", "d_out"))
        dot = ((g * w) * x).sum(-1) / case["width"]
        d_x = s["d_sum"].double() + g * w * inverse[:, None] - x * (inverse ** 3 * dot)[:, None]
        return dict(d_x=d_x, d_weight=inverse @ (g * x))
    if kind == "quantize":
        if case["transposed"]:
            return _rounded64(s["source"].t()).t().contiguous()
        return _rounded64(s["source"])
    if kind == "product":
        x = _values64(s["left_codes"], s["left_scales"], case["inner"])
        w = _values64(s["right_codes"], s["right_scales"], case["inner"])
        return x @ w.T.contiguous() + s["bias"].double()
    n, heads, classes = case["rows"], case["heads"], case["classes"]
    z = (s["logits"][:, case["offset"]:].double() * case["scale"]).view(n, heads, classes)
    log_p = z - torch.logsumexp(z, -1, keepdim=True)
    plogp = torch.where(torch.isinf(log_p), torch.zeros_like(z), torch.exp(log_p) * log_p)
    entropy = -plogp.sum(-1)
    given = s["tokens"] != EMPTY
    token = torch.where(given, s["tokens"], torch.zeros_like(s["tokens"])).long()[..., None]
    if kind == "logprobs":
        largest = s["logits"][:, case["offset"]:].view(n, heads, classes).amax(-1)
        log_total = torch.logsumexp(z, -1) - largest.double() * case["scale"]
        lp = torch.where(given, torch.take_along_dim(log_p, token, -1)[..., 0], torch.zeros_like(entropy))
        out = dict(logprobs=lp, entropies=entropy, stats=torch.stack([largest.double(), log_total], -1))
        if case["top"] == 0:
            return out
        left, index, best = z.clone(), torch.arange(classes, device="cuda"), []
        for _ in range(case["top"]):  # the largest left, at its lowest class
            at = torch.where(left == left.amax(-1, keepdim=True), index, classes).amin(-1, keepdim=True)
            best.append(at)
            left.scatter_(-1, at, -math.inf)
        best = torch.cat(best, -1)
        return dict(out, top_tokens=best.int(), top_logprobs=torch.take_along_dim(log_p, best, -1))
    p = torch.exp(log_p)
    d_lp = torch.where(given, s["d_logprobs"], torch.zeros_like(s["d_logprobs"])).double()[..., None]
    one_hot = torch.arange(classes, device="cuda") == token
    grad = d_lp * (one_hot.double() - p) - s["d_entropies"].double()[..., None] * (plogp + p * entropy[..., None])
    out = torch.zeros(s["logits"].shape, device="cuda", dtype=torch.float64)
    out[:, case["offset"]:] = case["scale"] * grad.flatten(1)
    return out
