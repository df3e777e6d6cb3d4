"""What is measured of the 4-bit layer: products with weights held in 4 bits, the root-mean-square norm in front of them, and
the step that makes such weights out of a matrix.

`listed()` and `draw()` give the cases, `prepare()` what a program holds before the call, `run()` one pass, `exact()` the same
from the definition in 64 bits.  With `own` false `run` computes with elementary torch operations, with `own` true it calls the
library's C ABI (include/decx_hip.h) on the tensors' addresses and the current stream.

4-bit weights, N x K in groups of 32, 64 or 128 along K: W(n, k) = (code - zero) * scale, zero = 8 where there are no zero points.
The codes lie in tiles of 16 rows x 128 columns, 1024 bytes each, [row tile][column tile]; in a tile the 32-bit word
[kg 0..3][row 0..15][j 0..3] holds columns 32 j + 8 kg + 0..7, in its nibbles 0, 4, 1, 5, 2, 6, 3, 7.  Scales (fp16) and zero
points (a byte each) lie [row tile][column tile][row 0..15][group of the tile]."""
import math

import torch

own = False

WORKSPACE_BYTES = 32 << 20


def listed():
    return [
        # one token against a square projection: the smallest call of a serving loop, latency counts
        {"name": "token_4096x4096_f16", "op": "product", "m": 1, "n": 4096, "k": 4096, "group": 128, "zeros": False, "x": "f16", "y": "f16", "c": 0},
        # one token, activations in 8 bits as the norm writes them, weights with zero points
        {"name": "token_8192x8192_i8", "op": "product", "m": 1, "n": 8192, "k": 8192, "group": 128, "zeros": True, "x": "i8", "y": "f16", "c": 0},
        # one token against the largest matrix of a model, the one onto its vocabulary: fp32 logits, fine groups
        {"name": "token_65536x8192_f16_g32", "op": "product", "m": 1, "n": 65536, "k": 8192, "group": 32, "zeros": False, "x": "f16", "y": "f32", "c": 0},
        # seven sequences decoded together, sizes that divide nothing, zero points, the residual added in the same call
        {"name": "batch_7_odd_f16_g64", "op": "product", "m": 7, "n": 5003, "k": 7001, "group": 64, "zeros": True, "x": "f16", "y": "f16", "c": 2},
        # sixty sequences decoded together, 8-bit activations
        {"name": "batch_60_i8", "op": "product", "m": 60, "n": 8192, "k": 4096, "group": 128, "zeros": False, "x": "i8", "y": "f16", "c": 0},
        # a ragged prompt in 8 bits, one bias row added
        {"name": "prompt_1000_i8_g64", "op": "product", "m": 1000, "n": 4096, "k": 8192, "group": 64, "zeros": True, "x": "i8", "y": "f16", "c": 1},
        # a long prompt: bound by the matrix cores
        {"name": "prompt_4096_f16", "op": "product", "m": 4096, "n": 8192, "k": 8192, "group": 128, "zeros": False, "x": "f16", "y": "f16", "c": 0},
        # the norm of one token: residual added and kept, 8 bits out
        {"name": "norm_1x4096_q8", "op": "norm", "rows": 1, "cols": 4096, "type": "f16", "residual": True, "sum": True, "out": "q8"},
        # the norm of a long prompt, the same form
        {"name": "norm_4096x8192_q8", "op": "norm", "rows": 4096, "cols": 8192, "type": "f16", "residual": True, "sum": True, "out": "q8"},
        # fp32 rows of an odd length, no residual, fp32 out
        {"name": "norm_777x5001_f32", "op": "norm", "rows": 777, "cols": 5001, "type": "f32", "residual": False, "sum": False, "out": "same"},
        # a square projection laid out once in 4 bits, and the values that stand for it
        {"name": "quantize_4096x4096_f16", "op": "quantize", "n": 4096, "k": 4096, "group": 128, "zeros": False, "type": "f16"},
        # fp32 weights of odd sizes with zero points in fine groups
        {"name": "quantize_5003x7001_f32_g32", "op": "quantize", "n": 5003, "k": 7001, "group": 32, "zeros": True, "type": "f32"},
    ]


def _log(rng, low, high):
    """A whole number from `low` to `high`, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _length(rng, low, high):
    """The same; half of them whole multiples of 64 where that fits, the others as they fall (odd ones among them)."""
    v = _log(rng, low, high)
    return max(64, v // 64 * 64) if v >= 64 and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["product", "product", "product", "norm", "quantize"])
    if op == "product":
        m = 1 if rng.random() < 0.3 else _log(rng, 1, 4096)
        n, k = _length(rng, 16, 65536), _length(rng, 32, 16384)
        while n * k > 65536 * 8192 or m * n * k > 4096 * 8192 * 8192:
            n = max(1, n // 2)
        return {"op": op, "m": m, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "x": rng.choice(["f16", "i8"]),
                "y": rng.choice(["f16", "f16", "f32"]), "c": rng.choice([0, 0, 1, 2])}
    if op == "norm":
        rows, cols = _log(rng, 1, 4096), _length(rng, 16, 40000)
        while rows * cols > 4096 * 8192:
            rows //= 2
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(["f16", "f16", "f32"]), "residual": rng.random() < 0.7, "sum": rng.random() < 0.7,
                "out": rng.choice(["q8", "q8", "same"])}
    n, k = _length(rng, 16, 16384), _length(rng, 32, 16384)
    while n * k > 8192 * 8192:
        n //= 2
    return {"op": op, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "type": rng.choice(["f16", "f32"])}


def _tiles(n, k):
    return -(-n // 16), -(-k // 128)


def _type(name):
    return {"f16": torch.float16, "f32": torch.float32}[name]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if case["op"] == "product":
        m, n, k, per_tile = case["m"], case["n"], case["k"], 128 // case["group"]
        nt, kt = _tiles(n, k)
        # codes as rounded normal weights leave them: most of them near the middle
        nibbles = (normal(nt, kt, 1024, 2) * 2.6 + 8).round_().clamp_(0, 15).to(torch.uint8)
        s["codes"] = nibbles[..., 0] | nibbles[..., 1] << 4
        s["scales"] = (normal(nt, kt, 16, per_tile).abs() * 0.002 + 0.004).half()
        s["zeros"] = torch.randint(4, 12, (nt, kt, 16, per_tile), generator=g, device="cuda").to(torch.uint8) if case["zeros"] else None
        x = normal(m, k) * (1 + 4 * (torch.rand(1, k, generator=g, device="cuda") < 0.01))     # a few channels stand out
        if case["x"] == "i8":
            top = x.abs().amax(1, keepdim=True).clamp_(min=1e-6)
            s["x"], s["x_scales"] = (x * 127 / top).round_().to(torch.int8), (top[:, 0] / 127).contiguous()
        else:
            s["x"], s["x_scales"] = x.half(), None
        out = _type(case["y"])
        s["c"] = normal(m if case["c"] == 2 else 1, n).to(out) if case["c"] else None
        s["alpha"], s["beta"] = (0.5, 1.0) if case["c"] else (1.0, 1.0)
        s["y"] = torch.empty(m, n, dtype=out, device="cuda")
        s["workspace"] = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    elif case["op"] == "norm":
        rows, cols, t = case["rows"], case["cols"], _type(case["type"])
        s["x"] = normal(rows, cols).to(t)
        # the residual stream: larger than what a layer adds to it, a few channels much larger
        s["residual"] = (normal(rows, cols) * (3 + 30 * (torch.rand(1, cols, generator=g, device="cuda") < 0.003))).to(t) if case["residual"] else None
        s["weight"] = (1 + normal(cols, scale=0.2)).to(t)
        s["sum"] = torch.empty(rows, cols, dtype=t, device="cuda") if case["sum"] else None
        s["y"] = torch.empty(rows, cols, dtype=torch.int8 if case["out"] == "q8" else t, device="cuda")
        s["y_scales"] = torch.empty(rows, device="cuda") if case["out"] == "q8" else None
    else:
        n, k, per_tile = case["n"], case["k"], 128 // case["group"]
        nt, kt = _tiles(n, k)
        s["w"] = (normal(n, k, scale=0.02) + (normal(n, 1, scale=0.01) if case["zeros"] else 0)).to(_type(case["type"]))
        s["codes"] = torch.empty(nt, kt, 1024, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(nt, kt, 16, per_tile, dtype=torch.float16, device="cuda")
        s["zeros"] = torch.empty(nt, kt, 16, per_tile, dtype=torch.uint8, device="cuda") if case["zeros"] else None
        s["values"] = torch.empty(n, k, device="cuda")
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _by_row(per_group, n):
    """[row tile][column tile][row][group] -> [row][group along K]."""
    return per_group.permute(0, 2, 1, 3).flatten(2).flatten(0, 1)[:n]


def _plain_weights(s, n, k, group):
    words = s["codes"].view(torch.int32).view(*s["codes"].shape[:2], 4, 16, 4, 1)
    nibble = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device="cuda")
    q = (words >> nibble) & 15                                                   # [row tile][column tile][kg][row][j][8]
    q = q.permute(0, 3, 1, 4, 2, 5).reshape(words.shape[0] * 16, -1)[:n].float()  # [row][column]
    q = q.view(n, -1, group)
    q = q - (_by_row(s["zeros"], n).float()[..., None] if s["zeros"] is not None else 8.0)
    return (q * _by_row(s["scales"], n).float()[..., None]).view(n, -1)[:, :k]


def _plain_product(s, case):
    w = _plain_weights(s, case["n"], case["k"], case["group"])
    y = s["x"].float() @ w.t()
    if s["x_scales"] is not None:
        y = y * s["x_scales"][:, None]
    if s["c"] is not None:
        y = s["alpha"] * y + s["beta"] * s["c"].float()
    return y.to(s["y"].dtype)


def _plain_norm(s, case):
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    wide = h.float() if case["type"] == "f16" else h.double()                     # products of two fp16 are whole in fp32, those of two fp32 in 64 bits
    rho = 1 / torch.sqrt(wide.square().mean(1, keepdim=True) + 1e-5)
    t = wide * s["weight"].to(wide.dtype)
    kept = h if case["sum"] else None
    if case["out"] != "q8":
        return {"sum": kept, "y": (t * rho).to(h.dtype)}
    top = t.abs().amax(1, keepdim=True)
    codes = torch.round(127 * t.double() / top.double())                          # 64 bits: values next to a border
    return {"sum": kept, "codes": torch.where(top > 0, codes, 0.0).to(torch.int8), "scales": (top * rho / 127).float()[:, 0]}


def _plain_quantize(s, case):
    n, k, group = case["n"], case["k"], case["group"]
    w = torch.nn.functional.pad(s["w"].float(), (0, -k % group)).view(n, -1, group)
    if case["zeros"]:
        low, high = w.amin(2, keepdim=True).clamp(max=0), w.amax(2, keepdim=True).clamp(min=0)
        scale = ((high - low) / torch.full_like(low, 15.0)).half().double()         # (a plain number as divisor would become a product)
        zero = torch.where(scale > 0, torch.round(-low.double() / scale).clamp(0, 15), 8.0)
    else:
        top = w.abs().amax(2, keepdim=True)
        scale = (top / torch.full_like(top, 7.0)).half().double()
        zero = torch.full_like(scale, 8.0)
    q = torch.where(scale > 0, (torch.round(w.double() / scale) + zero).clamp(0, 15), zero)
    return ((q - zero) * scale).float().view(n, -1)[:, :k].contiguous()


# ---- the library's calls ---------------------------------------------------------------------------------------------

_lib = None


def _library():
    global _lib
    if _lib is None:
        from decx_amd import hip
        hip.init(0)
        _lib = hip.lib()
    return _lib


def _at(t):
    return t.data_ptr() if t is not None else None


def _done(rc):
    if rc != 0:
        raise RuntimeError("the library refused the call: %d" % rc)


def _own_product(s, case):
    L = _library()
    m, n, k = case["m"], case["n"], case["k"]
    rest = (_at(s["codes"]), _at(s["scales"]), _at(s["zeros"]), _at(s["c"]), _at(s["y"]), m, n, k, case["group"], k, n if case["c"] == 2 else 0, n,
            s["alpha"], s["beta"], 1 if case["y"] == "f32" else 0, _at(s["workspace"]), WORKSPACE_BYTES, s["stream"])
    if case["x"] == "i8":
        _done(L.decx_hip_gemm_q4_i8(_at(s["x"]), _at(s["x_scales"]), *rest))
    else:
        _done(L.decx_hip_gemm_q4_f16(_at(s["x"]), *rest))
    return s["y"]


def _own_norm(s, case):
    L = _library()
    rows, cols, q8 = case["rows"], case["cols"], case["out"] == "q8"
    call = L.decx_hip_rmsnorm_f16 if case["type"] == "f16" else L.decx_hip_rmsnorm_f32
    _done(call(_at(s["x"]), _at(s["residual"]), _at(s["weight"]), _at(s["sum"]), _at(s["y"]), _at(s["y_scales"]), rows, cols, cols,
               cols if case["residual"] else 0, cols if case["sum"] else 0, cols, 1e-5, s["stream"]))
    return {"sum": s["sum"], "codes": s["y"], "scales": s["y_scales"]} if q8 else {"sum": s["sum"], "y": s["y"]}


def _own_quantize(s, case):
    L = _library()
    n, k, group = case["n"], case["k"], case["group"]
    call = L.decx_hip_q4_quantize_f16 if case["type"] == "f16" else L.decx_hip_q4_quantize_f32
    _done(call(_at(s["w"]), _at(s["codes"]), _at(s["scales"]), _at(s["zeros"]), n, k, k, group, s["stream"]))
    _done(L.decx_hip_q4_dequantize_f32(_at(s["codes"]), _at(s["scales"]), _at(s["zeros"]), _at(s["values"]), n, k, k, group, s["stream"]))
    return s["values"]


def run(state):
    case = state["case"]
    if own:
        return {"product": _own_product, "norm": _own_norm, "quantize": _own_quantize}[case["op"]](state, case)
    return {"product": _plain_product, "norm": _plain_norm, "quantize": _plain_quantize}[case["op"]](state, case)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def _exact_rows(s, n0, n1, k, group):
    """Rows n0..n1-1 of the weights: every code fetched from the place that the layout gives it."""
    per_tile, kt = 128 // group, s["codes"].shape[1]
    row = torch.arange(n0, n1, device="cuda")[:, None]
    col = torch.arange(k, device="cuda")[None, :]
    inside = col % 128
    word = (((row // 16 * kt + col // 128) * 4 + inside % 32 // 8) * 16 + row % 16) * 4 + inside // 32
    place = inside % 8 // 2 + inside % 2 * 4
    byte = s["codes"].flatten()[word * 4 + place // 2].long()
    code = torch.where(place % 2 == 1, byte // 16, byte % 16).double()
    at = ((row // 16 * kt + col // 128) * 16 + row % 16) * per_tile + inside // group
    zero = 8.0 if s["zeros"] is None else s["zeros"].flatten()[at].double()
    return (code - zero) * s["scales"].flatten()[at].double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        n, k = case["n"], case["k"]
        x = s["x"].double()
        if s["x_scales"] is not None:
            x = x * s["x_scales"].double()[:, None]
        step = max(16, (1 << 27) // max(1, k))
        y = torch.cat([torch.mm(x, _exact_rows(s, at, min(n, at + step), k, case["group"]).t().contiguous()) for at in range(0, n, step)], 1)
        return y if s["c"] is None else s["alpha"] * y + s["beta"] * s["c"].double()
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = (h + s["residual"].double()).to(s["x"].dtype).double()            # the sum is held in the rows' type
        kept = h if case["sum"] else None
        y = h * s["weight"].double() / (h.pow(2).sum(1, keepdim=True) / case["cols"] + 1e-5).sqrt()
        if case["out"] != "q8":
            return {"sum": kept, "y": y}
        scale = y.abs().amax(1) / 127
        t = h * s["weight"].double()
        codes = (t * 127 / t.abs().amax(1, keepdim=True)).nan_to_num(0.0).round().to(torch.int8)
        return {"sum": kept, "codes": codes, "scales": scale}
    n, k, group = case["n"], case["k"], case["group"]
    out = torch.empty(n, k, dtype=torch.float64, device="cuda")
    for at in range(0, k, group):
        w = s["w"][:, at:at + group].double()
        low, high = w.min(1, keepdim=True).values.clamp(max=0), w.max(1, keepdim=True).values.clamp(min=0)
        if case["zeros"]:
            step = ((high - low).float().double() / torch.full_like(low, 15.0)).float().half().double()   # by definition in fp32, held in fp16
            zero = torch.where(step > 0, (-low / step).round().clamp(0, 15), 8.0)
        else:
            step = (torch.maximum(high, -low) / torch.full_like(low, 7.0)).float().half().double()
            zero = torch.full_like(step, 8.0)
        code = torch.where(step > 0, ((w / step).round() + zero).clamp(0, 15), zero)
        out[:, at:at + group] = (code - zero) * step
    return out


def work(case):
    """Each input read once, each output written once."""
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        groups, out = -(-k // case["group"]), 4 if case["y"] == "f32" else 2
        weights = n * -(-k // 2) + n * groups * (3 if case["zeros"] else 2)
        x = m * k * 2 if case["x"] == "f16" else m * k + 4 * m
        return {"bytes": weights + x + m * n * out + (0, n, m * n)[case["c"]] * out, "flops": 2 * m * n * k}
    if case["op"] == "norm":
        size, b = case["rows"] * case["cols"], 2 if case["type"] == "f16" else 4
        out = size + 4 * case["rows"] if case["out"] == "q8" else size * b
        return {"bytes": size * b * (1 + case["residual"] + case["sum"]) + case["cols"] * b + out, "flops": 8 * size}
    n, k = case["n"], case["k"]
    packed = n * -(-k // 2) + n * -(-k // case["group"]) * (3 if case["zeros"] else 2)
    return {"bytes": n * k * (2 if case["type"] == "f16" else 4) + 2 * packed + 4 * n * k, "flops": 6 * n * k}
