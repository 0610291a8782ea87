"""The products of `paracel_b200.ops.grouped` and `paracel_b200.ops.mx4`: cases, inputs, plain forms and values in 64 bits.

Grouped products: rows of X sorted by the expert that works on them (segment, cluster, user group: whatever the
rows are routed by), expert e's rows in [offsets[e], offsets[e + 1]), one matrix W[e] (N x K) for each.
    nt     Y[t]  = W[e] x[t]                    the layer's values
    step   nt, and its gradients dX[t] = W[e]^T dY[t] and dW[e] = sum over its rows of dY[t] x[t]^T
Four-bit microscaled matrices: blocks of 32 values along a row share a power of two (8 bits, 2^(code - 127)); a value
is one of 0, .5, 1, 1.5, 2, 3, 4, 6 and a sign. Two of them share a byte, the first in the low half: data[r, K/2];
scales[b, r, i] is the code of row r's block 4 b + i.
    quantize   x to blocks and back: the values that the four bits stand for
    mx4        Y = x q^T: x is quantised in the call, q is kept in four bits
    mx4_group  the same with one matrix for each expert

`own` says which side runs: False, elementary torch operations in 32 bits; True, the calls of the package.
"""
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one step of a few users over many experts: latency, and the weights of the experts that have a row
        dict(name="nt_decode", op="nt", type="bf16", E=32, T=16, N=1536, K=1024, spare=0),
        # sizes that divide by nothing, a padded batch (rows behind the last expert's)
        dict(name="nt_odd", op="nt", type="fp16", E=11, T=1537, N=1001, K=776, spare=13),
        # a large batch through wide experts
        dict(name="nt_large", op="nt", type="bf16", E=32, T=32768, N=4096, K=2048, spare=0),
        # training: the layer's values and both gradients
        dict(name="step_small", op="step", type="fp16", E=24, T=1000, N=520, K=264, spare=0),
        dict(name="step_large", op="step", type="bf16", E=16, T=16384, N=2048, K=1024, spare=0),
        # a batch of factor rows, an odd number of columns; and a table of half a gigabyte
        dict(name="quantize_small", op="quantize", type="fp32", T=257, K=100),
        dict(name="quantize_large", op="quantize", type="bf16", T=32768, K=8192),
        # one query against a table in four bits, a ragged batch, a large one
        dict(name="mx4_single", op="mx4", type="bf16", T=1, N=8192, K=4096),
        dict(name="mx4_odd", op="mx4", type="fp16", T=301, N=1001, K=1000),
        dict(name="mx4_large", op="mx4", type="bf16", T=8192, N=8192, K=8192),
        # experts served from four bits: a few rows, and a large batch
        dict(name="mx4_group_decode", op="mx4_group", type="bf16", E=64, T=24, N=2048, K=2048, spare=0),
        dict(name="mx4_group_large", op="mx4_group", type="bf16", E=32, T=16384, N=4096, K=2048, spare=0),
    ]


def draw(rng):
    def log(lo, hi, step=1):
        v = int(round(lo * (hi / lo) ** rng.random()))
        return min(hi, max(lo, v // step * step))

    op = rng.choice(("nt", "step", "quantize", "mx4", "mx4_group"))
    odd = rng.random() < 0.3
    c = dict(op=op, type=rng.choice(("bf16", "fp16")))
    if op == "quantize":
        c.update(type=rng.choice(("bf16", "fp16", "fp32")), T=log(1, 32768), K=log(33, 8192, 1 if odd else 8))
        return c
    if op == "mx4":
        c.update(T=log(1, 8192), N=log(64, 8192, 1 if odd else 8), K=log(64, 8192, 1 if odd else 32))
        return c
    c.update(E=log(1, 64), T=log(1, 32768 if op == "nt" else 16384), N=log(64, 4096 if op != "step" else 2048, 1 if odd else 8),
             K=log(64, 2048 if op != "step" else 1024, 1 if odd else 8), spare=rng.choice((0, 0, rng.randrange(1, 40))))
    c["E"] = max(1, min(c["E"], (32 * 4096 * 2048) // (c["N"] * c["K"])))
    return c


# ------------------------------------------------------------------------------------------------ inputs

def _rows(n, k, dtype, g):
    """Rows as activations are: normal values, some columns larger than the others, a row of zeros now and then."""
    x = torch.randn(n, k, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))
    x *= (torch.rand(n, 1, device="cuda", generator=g) > 0.01)
    return x.to(dtype)


def _offsets(E, T, seed):
    """Where each expert's rows begin: shares spread by a factor of about e either way, some of them empty when rows are few."""
    g = torch.Generator().manual_seed(seed)
    share = torch.exp(0.5 * torch.randn(E, generator=g))
    to = torch.multinomial(share, T, replacement=True, generator=g)
    counts = torch.bincount(to, minlength=E)
    off = torch.zeros(E + 1, dtype=torch.int32)
    off[1:] = counts.cumsum(0)
    return off.cuda(), int(counts.max())


def _pack(w):
    """(data, scales) of w's rows in four bits, laid out as the package keeps them."""
    rows, k = w.shape
    code, sign, e = _codes(w)
    code = (code + 8 * sign).to(torch.uint8).view(rows, -1, 2)
    data = code[..., 0] + 16 * code[..., 1]
    blocks = e.shape[1]
    scales = torch.zeros((blocks + 3) // 4 * 4, rows, dtype=torch.uint8, device=w.device)
    scales[:blocks] = (e + 127).to(torch.uint8).T
    return data.contiguous(), scales.view(-1, 4, rows).transpose(1, 2).contiguous()


def prepare(case, seed):
    c = dict(case, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[c["type"]]
    s = dict(op=c["op"], type=t, K=c["K"])
    if c["op"] == "quantize":
        s["x"] = _rows(c["T"], c["K"], t, g)
        return s
    E = c.get("E", 1)
    s.update(E=E, N=c["N"], x=_rows(c["T"] + c.get("spare", 0), c["K"], t, g))
    w = torch.randn(E * c["N"], c["K"], device="cuda", generator=g) / c["K"] ** 0.5
    if c["op"].startswith("mx4"):
        s["data"], s["scales"] = _pack(w)
    else:
        s["w"] = w.to(t).view(E, c["N"], c["K"])
    if "E" in c:
        s["offsets"], s["longest"] = _offsets(E, c["T"], seed)
    if c["op"] == "step":
        s["dy"] = _rows(c["T"] + c["spare"], c["N"], t, g)
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _blocks(x):
    """x in 32 bits as [rows, blocks, 32], the last block filled up with zeros."""
    rows, k = x.shape
    y = torch.zeros(rows, (k + 31) // 32 * 32, device=x.device)
    y[:, :k] = x
    return y.view(rows, -1, 32)


def _codes(x):
    """(index into VALUES, sign, exponent of each block) of x's values; the largest of a block is below 8 after scaling."""
    b = _blocks(x)
    most = b.abs().amax(2)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -127).clamp(-127, 127)
    v = torch.ldexp(b.abs(), -e[..., None])
    code = ((v > 0.25).int() + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5))
    return code, (b < 0).int(), e


def _quantized(x):
    """What x's four bits stand for, in 32 bits, [rows, blocks, 32]."""
    b = _blocks(x)
    most = b.abs().amax(2, keepdim=True)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -127).clamp(-127, 127)
    v = torch.ldexp(b, -e)
    step = 0.5 + 0.5 * (v.abs() >= 2) + (v.abs() >= 4)
    return torch.ldexp((torch.round(v / step) * step).clamp(-6, 6), e)


def _unpacked(data, scales, rows):
    """The values of a packed matrix, in 32 bits, [rows, blocks * 32]."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=data.device)
    v = torch.stack((table[(data & 15).long()], table[(data >> 4).long()]), 2).view(rows, -1, 32)
    e = scales.transpose(1, 2).reshape(-1, rows)[: v.shape[1]].T.int() - 127
    return torch.ldexp(v, e[..., None]).view(rows, -1)


def _spread(s, x):
    """x's rows as [experts, longest, columns] in 32 bits, zeros behind an expert's last row; and which places are taken."""
    at = torch.arange(s["longest"], device=x.device)
    begin, end = s["offsets"][:-1, None], s["offsets"][1:, None]
    taken = begin + at < end
    row = (begin + at).clamp(max=x.shape[0] - 1).long()
    return torch.where(taken[..., None], x[row].float(), 0.0), taken, row


def _gathered(y, taken, row, rows, dtype):
    out = torch.zeros(rows, y.shape[2], dtype=dtype, device=y.device)
    out[row[taken]] = y[taken].to(dtype)
    return out


def _plain(s):
    x, t = s["x"], s["type"]
    if s["op"] == "quantize":
        return _quantized(x).view(x.shape[0], -1)[:, : s["K"]].to(torch.bfloat16)
    if s["op"] == "mx4":
        q = _unpacked(s["data"], s["scales"], s["N"])
        return (_quantized(x).view(x.shape[0], -1) @ q.T).to(t)
    if s["op"] == "mx4_group":
        q = _unpacked(s["data"], s["scales"], s["E"] * s["N"]).view(s["E"], s["N"], -1)
        xs, taken, row = _spread(s, _quantized(x).view(x.shape[0], -1))
        return _gathered(torch.bmm(xs, q.transpose(1, 2)), taken, row, x.shape[0], t)
    w = s["w"].float()
    xs, taken, row = _spread(s, x)
    y = _gathered(torch.bmm(xs, w.transpose(1, 2)), taken, row, x.shape[0], t)
    if s["op"] == "nt":
        return y
    ds = _spread(s, s["dy"])[0]
    dx = _gathered(torch.bmm(ds, w), taken, row, x.shape[0], t)
    return y, dx, torch.bmm(ds.transpose(1, 2), xs).to(t)


# ------------------------------------------------------------------------------------------------ the package's calls

def _own(s):
    x = s["x"]
    if s["op"] == "quantize":
        from paracel_b200.ops.mx4 import mx4_dequantize, mx4_quantize
        return mx4_dequantize(mx4_quantize(x), torch.bfloat16)
    if s["op"] == "mx4":
        from paracel_b200.ops.mx4 import Mx4Matrix, mx4_gemm_nt
        return mx4_gemm_nt(x, Mx4Matrix(s["data"], s["scales"], s["K"]))
    if s["op"] == "mx4_group":
        from paracel_b200.ops.mx4 import Mx4Matrix, mx4_grouped_nt
        return mx4_grouped_nt(x, Mx4Matrix(s["data"], s["scales"], s["K"]), s["offsets"])
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    y = grouped_nt(x, s["w"], s["offsets"])
    if s["op"] == "nt":
        return y
    return y, grouped_nn(s["dy"], s["w"], s["offsets"]), grouped_tn(s["dy"], x, s["offsets"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ work and 64 bits

def work(case):
    c, size = case, 4 if case["type"] == "fp32" else 2
    T, K = c["T"], c["K"]
    if c["op"] == "quantize":
        return {"bytes": T * K * (size + 2), "flops": 0}
    N, E = c["N"], c.get("E", 1)
    # experts that have a row: only their matrices are read (the expectation for equal shares)
    used = E * (1 - (1 - 1 / E) ** T) if E > 1 else 1
    weights = used * N * K * (17 / 32 if c["op"].startswith("mx4") else 2)
    if c["op"] == "step":
        # x, dy, w in; y, dx and every dw out
        return {"bytes": weights + 2 * (2 * T * K + 2 * T * N) + 2 * E * N * K, "flops": 6 * T * N * K}
    return {"bytes": weights + 2 * (T * K + T * N), "flops": 2 * T * N * K}


def _nearest(x):
    """Every block of 32 of x's rows divided by 2^(floor(log2 of its largest) - 2) and rounded to the nearest of the eight
    magnitudes, the even one of the two at a tie, in 64 bits."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -k % 32)).reshape(-1, 32)
    grid = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    most = x.abs().max(1, keepdim=True).values
    top = torch.exp2(torch.round(torch.log2(most.clamp(min=2.0 ** -160))))  # a power of two next to the largest
    top = torch.where(top > most, top / 2, top)  # the one at or below it: a logarithm may be off in its last bit
    scale = (top / 4).clamp(min=2.0 ** -127)
    v = (x / scale).abs().clamp(max=6.0)
    up = torch.searchsorted(grid, v).clamp(max=7)
    down = (up - 1).clamp(min=0)
    a, b = v - grid[down], grid[up] - v
    pick = torch.where(a < b, down, torch.where(b < a, up, torch.where(down % 2 == 0, down, up)))
    return (torch.sign(x) * grid[pick] * scale).view(rows, -1)[:, :k]


def _kept(s, rows):
    """The packed matrix in 64 bits: the two halves of a byte, looked up, times two to the scale's code less 127."""
    lut = torch.tensor(VALUES, dtype=torch.float64, device="cuda")
    out = torch.empty(rows, s["data"].shape[1] * 2, dtype=torch.float64, device="cuda")
    for half in (0, 1):
        code = (s["data"] >> (4 * half)) & 15
        out[:, half::2] = lut[(code & 7).long()] * (1.0 - 2.0 * (code >> 3))
    for b in range(out.shape[1] // 32):
        out[:, 32 * b:32 * b + 32] *= torch.exp2(s["scales"][b // 4, :, b % 4].double() - 127)[:, None]
    return out[:, : s["K"]]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if s["op"] == "quantize":
        return _nearest(x)
    if s["op"] == "mx4":
        return _nearest(x) @ _kept(s, s["N"]).T
    if s["op"] == "mx4_group":
        x, w = _nearest(x), _kept(s, s["E"] * s["N"]).view(s["E"], s["N"], -1)
    else:
        w = s["w"].double()
    off = s["offsets"].tolist()
    y = torch.zeros(x.shape[0], s["N"], dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros(s["E"], s["N"], s["K"], dtype=torch.float64, device="cuda")
    for e in range(s["E"]):
        lo, hi = off[e], off[e + 1]
        y[lo:hi] = x[lo:hi] @ w[e].T
        if s["op"] == "step":
            d = s["dy"][lo:hi].double()
            dx[lo:hi] = d @ w[e]
            dw[e] = d.T @ x[lo:hi]
    return (y, dx, dw) if s["op"] == "step" else y
