"""Four-bit microscaled matrices against their definition in 64 bits.

A product of two four-bit values and their scales is exact in fp32 as long as nothing leaves its range; the sum of K of them is off by at most
one unit in the last of 24 bits of a partial sum (at most S = sum |a| |b|) for each addition, K 2^-23 S, and by half a step of the
result's type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BF, FP, F = torch.bfloat16, torch.float16, torch.float32


def _define(x):
    """What the format keeps of x [rows, K], in 64 bits: every block of 32 divided by its scale, the nearest value of the grid."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(rows, -1, 32)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    most = b.abs().amax(2, keepdim=True)
    exponent = torch.frexp(torch.where(torch.isfinite(most) & (most > 0), most, 2.0 ** -140)).exponent - 3
    scale = torch.ldexp(torch.ones_like(most), exponent.clamp(min=-127))
    v = (b / scale).abs().clamp(max=6.0)
    away = (v[..., None] - grid).abs()                       # ties: of two neighbours at the same distance the even code
    best = away.amin(-1, keepdim=True)
    even = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)
    at = (away[..., even] == best).int().argmax(-1)
    q = torch.sign(b) * grid[even[at]] * scale
    q = torch.where(torch.isfinite(most), q, torch.nan)
    return q.view(rows, -1)[:, :k]


def _rows(rows, k, dtype=F, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, device="cuda", generator=g) * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))
    return x.to(dtype)


def _same(a, b):
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    assert torch.equal(torch.nan_to_num(a.double(), nan=0.0), torch.nan_to_num(b.double(), nan=0.0))


@pytest.mark.parametrize("dtype", [F, BF, FP])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (5, 33), (33, 100), (64, 128), (31, 129), (257, 777), (1000, 1024),
                                    (2, 4100), (70, 2048)])
def test_quantisation_is_the_formats(rows, k, dtype):
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_quantize
    x = _rows(rows, k, dtype)
    q = mx4_quantize(x)
    want = _define(x)
    _same(mx4_dequantize(q), want)
    _same(mx4_dequantize(q, BF), want)
    _same(mx4_dequantize(q, FP), want.to(F).to(FP))
    # the layout that the class documents
    table = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device="cuda")
    codes = torch.stack((q.data & 15, q.data >> 4), 2).view(rows, -1)
    scales = q.scales.transpose(1, 2).reshape(-1, rows).T[:, :codes.shape[1] // 32]
    v = table[codes.long()].view(rows, -1, 32) * torch.exp2(scales.double() - 127)[..., None]
    _same(v.view(rows, -1)[:, :k], want)
    assert not codes[:, k:].any()
    assert not q.scales.transpose(1, 2).reshape(-1, rows)[codes.shape[1] // 32:].any()
    assert q.rows == rows and q.cols == k and q.nbytes() == q.data.numel() + q.scales.numel()


def test_every_tie_and_border():
    """Blocks led by 4, so that the scale is one: every tie, its neighbours on both sides, and what is beyond 6."""
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_quantize
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9999995], device="cuda")
    v = torch.cat((ties, torch.nextafter(ties, ties * 0), torch.nextafter(ties, ties * 0 + 7.9999995), ties * 0, ties * 0 - 0.0))
    v = torch.cat((v, -v))
    x = torch.zeros(v.numel(), 32, device="cuda")
    x[:, 0], x[:, 7] = 4.0, v
    got = mx4_dequantize(mx4_quantize(x))
    _same(got, _define(x))
    assert got[0, 7] == 0 and got[1, 7] == 1 and got[2, 7] == 1 and got[3, 7] == 2 and got[4, 7] == 2 and got[5, 7] == 4 \
        and got[6, 7] == 4 and got[7, 7] == 6 and got[8, 7] == 6 and got[9, 7] == 6


def test_every_exponent_subnormals_and_what_is_not_a_number():
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_quantize
    e = torch.arange(-149, 128, device="cuda")
    lead = torch.ldexp(torch.ones(e.numel(), device="cuda", dtype=torch.float64), e).to(F)
    assert torch.all(lead > 0)
    x = lead[:, None] * torch.tensor([1.0, 0.1, -0.3, 0.55, 0.7, -0.9, 0.0, 1.9], device="cuda").repeat(8)[None]
    x = x.double().clamp(-3.4e38, 3.4e38).to(F)
    q = mx4_quantize(x)
    _same(mx4_dequantize(q), _define(x))
    _same(mx4_dequantize(q, BF), _define(x))
    assert int(q.scales.max()) <= 252
    y = _rows(6, 96)
    y[0, 3], y[1, 40], y[2, 95], y[3, 0] = float("nan"), float("inf"), float("-inf"), 3.4028234e38
    y[4], y[5, 32:64] = 0.0, 0.0
    got = mx4_dequantize(mx4_quantize(y))
    _same(got, _define(y))
    assert torch.isnan(got[0, :32]).all() and torch.isnan(got[1, 32:64]).all() and not torch.isnan(got[:, :32][1:]).any()


def test_quantising_strided_rows_and_stacks():
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_quantize
    big = _rows(50, 300, BF)
    for x in (big[:, 8:208], big[:, 3:203], big[:, ::2], big[::3], big[:1].expand(7, 300), big.T):
        _same(mx4_dequantize(mx4_quantize(x)), _define(x))
    w = _rows(60, 72, F).view(5, 12, 72)
    q = mx4_quantize(w)
    assert q.rows == 60
    _same(mx4_dequantize(q), _define(w.view(60, 72)))
    _same(mx4_dequantize(mx4_quantize(w[:, ::2, 1:66])), _define(w[:, ::2, 1:66].reshape(30, 65)))
    wide = torch.full((60, 90), 3.0, device="cuda", dtype=BF)
    mx4_dequantize(q, BF, out=wide[:, 5:77])
    _same(wide[:, 5:77], _define(w.view(60, 72)))
    assert torch.all(wide[:, :5] == 3) and torch.all(wide[:, 77:] == 3)
    assert mx4_quantize(torch.empty(0, 40, device="cuda")).rows == 0
    assert mx4_dequantize(mx4_quantize(torch.empty(0, 40, device="cuda"))).shape == (0, 40)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("E,N,K", [(5, 1, 64), (9, 1, 100), (300, 1, 1056), (1, 7, 96), (6, 5, 1), (4, 1, 1), (1, 1, 40)])
def test_stacks_with_a_dimension_of_one(E, N, K, dtype):
    """Such a dimension may report any stride, and the stack still counts as contiguous: rows lie K values apart all the same."""
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_grouped_nt, mx4_quantize
    big = _rows(max(E, N) * E * N, K, dtype)              # as far as any of these strides would lead
    w = big[:E * N].view(N, E, K).transpose(0, 1) if N == 1 else big[:E * N].view(E, N, K)
    odd = big.as_strided((E, N, K), (K * N, K if N > 1 else K * E, 1 if K > 1 else 7))
    want = _define(big[:E * N])
    for x in (w, odd, odd.clone()):
        assert x.shape == (E, N, K) and x.is_contiguous()
        q = mx4_quantize(x)
        assert q.rows == E * N and q.cols == K
        _same(mx4_dequantize(q), want)
        _same(mx4_dequantize(mx4_quantize(x[:, 0])), _define(x[:, 0]))
    A, kept = _grid(E, K, 3), _grid(big.shape[0], K, 4)
    got = mx4_grouped_nt(A, mx4_quantize(kept.as_strided(odd.shape, odd.stride())), torch.arange(E + 1, device="cuda"))
    assert torch.equal(got.double(), torch.stack([A[e].double() @ kept[e * N:(e + 1) * N].double().T for e in range(E)]))


def _near(got, a, b):
    """got against a @ b.T of the values that the four bits stand for."""
    a, b = a.double(), b.double()
    ref, mags = a @ b.T, a.abs() @ b.abs().T
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + a.shape[1] * 2.0 ** -23 * mags * (1 + 2.0 ** -8)
    if got.dtype == FP:
        tol += 2.0 ** -25
    off = (got.double() - ref).abs()
    assert torch.all(off <= tol), f"worst {float((off - tol).max())} beyond, at {int((off - tol).argmax())} of {off.numel()}"


def _grid(rows, k, seed):
    """Values of the grid, a 6 in each block (so its scale is one), times a power of two for each row: quantisation keeps them, and sums
    of products are exact in fp32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.tensor(GRID, device="cuda")[torch.randint(0, 8, (rows, k), device="cuda", generator=g)]
    v *= torch.randint(0, 2, (rows, k), device="cuda", generator=g) * 2.0 - 1
    v[:, ::32] = 6.0
    return v * torch.exp2(torch.randint(-3, 4, (rows, 1), device="cuda", generator=g).float())


PRODUCTS = [(1, 1, 1), (1, 8, 32), (1, 128, 64), (1, 4096, 512), (2, 130, 33), (7, 1000, 100), (8, 256, 256), (17, 129, 257), (64, 64, 1024),
            (100, 200, 300), (129, 127, 511), (256, 384, 768), (300, 1001, 1000), (513, 260, 2050), (1000, 640, 96),
            # a cluster for a tile; tiles of as many rows as an accumulator holds
            (1, 300, 2100), (64, 129, 4000), (33, 1000, 2048), (3000, 2500, 520), (2113, 4000, 300), (1700, 3333, 2049)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_products_of_the_grids_values_are_exact(M, N, K):
    from paracel_b200.ops.mx4 import check_status, mx4_gemm_nt, mx4_quantize
    A, B = _grid(M, K, 1), _grid(N, K, 2)
    got = mx4_gemm_nt(A, mx4_quantize(B))
    check_status()
    assert got.dtype == F
    assert torch.equal(got.double(), A.double() @ B.double().T)


@pytest.mark.parametrize("dtype", [F, BF, FP])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_products_match(M, N, K, dtype):
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_gemm_nt, mx4_quantize
    A, B = _rows(M, K, dtype, 3), _rows(N, K, dtype, 4) / 8
    qa, qb = mx4_quantize(A), mx4_quantize(B)
    got = mx4_gemm_nt(A, qb)
    assert got.dtype == dtype
    _near(got, mx4_dequantize(qa), mx4_dequantize(qb))
    assert torch.equal(mx4_gemm_nt(qa, qb, out_dtype=dtype), got)
    wide = torch.full((M, N + 9), 5.0, device="cuda", dtype=dtype)
    mx4_gemm_nt(qa, qb, out=wide[:, 4:-5])
    assert torch.equal(wide[:, 4:-5], got) and torch.all(wide[:, :4] == 5) and torch.all(wide[:, -5:] == 5)


def test_far_scales():
    """Scales at both ends of their range meet so that products stay in fp32's; a block that is not a number makes its row so and no other."""
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_gemm_nt, mx4_quantize
    A, B = _grid(40, 96, 5) * 2.0 ** -100, _grid(70, 96, 6) * 2.0 ** 100
    assert torch.equal(mx4_gemm_nt(A, mx4_quantize(B)).double(), A.double() @ B.double().T)
    A, B = _grid(40, 96, 5) * 2.0 ** 118, _grid(70, 96, 6) * 2.0 ** -110
    assert torch.equal(mx4_gemm_nt(A, mx4_quantize(B)).double(), A.double() @ B.double().T)
    A, B = _rows(200, 130), _rows(70, 130)
    A[3, 129], A[150, 0], B[11, 64] = float("nan"), float("inf"), float("nan")
    got = mx4_gemm_nt(A, mx4_quantize(B))
    nan = torch.zeros(200, 70, dtype=torch.bool, device="cuda")
    nan[3], nan[150], nan[:, 11] = True, True, True
    assert torch.equal(torch.isnan(got), nan)
    # codes of blocks that a row does not have are not looked at
    q = mx4_quantize(_grid(40, 96, 5))
    q.scales[0, :, 3] = 255
    assert torch.equal(mx4_gemm_nt(q, mx4_quantize(_grid(70, 96, 6))).double(), _grid(40, 96, 5).double() @ _grid(70, 96, 6).double().T)
    assert torch.equal(mx4_dequantize(q), _grid(40, 96, 5))


GROUPS = [([1], 0, 1, 1), ([0, 1, 0], 0, 33, 40), ([0, 0], 5, 40, 32), ([7, 0, 9], 0, 130, 65), ([16, 31, 33, 1], 3, 72, 200),
          ([127, 129, 255, 257], 1, 257, 130), ([300, 0, 0, 1, 511], 17, 520, 264), ([5] * 100, 0, 100, 100), ([0] * 63 + [70], 0, 136, 328),
          ([2, 260, 3], 0, 128, 1056), ([1500, 40], 0, 384, 512),
          ([3, 0, 1], 2, 256, 2100), ([33, 64], 0, 130, 4096), ([700, 0, 1300, 33, 208], 5, 2500, 288), ([257, 15, 1000, 0, 500, 470, 60], 0, 3333, 520)]


@pytest.mark.parametrize("counts,spare,N,K", GROUPS)
def test_grouped_products_are_exact(counts, spare, N, K):
    from paracel_b200.ops.mx4 import check_status, mx4_grouped_nt, mx4_quantize
    E, T = len(counts), sum(counts) + spare
    A, B = _grid(T, K, 1), _grid(E * N, K, 2).view(E, N, K)
    off = torch.tensor([0] + counts, device="cuda").cumsum(0)
    ref = torch.zeros(T, N, dtype=torch.float64, device="cuda")
    for e in range(E):
        ref[off[e]:off[e + 1]] = A[off[e]:off[e + 1]].double() @ B[e].double().T
    q = mx4_quantize(B)
    for o in (off, off.int()):
        assert torch.equal(mx4_grouped_nt(A, q, o).double(), ref)
    kept = torch.full((T, N), 9.0, device="cuda", dtype=BF)
    mx4_grouped_nt(A, q, off, out=kept)
    n = sum(counts)
    assert torch.equal(kept[:n], ref[:n].to(BF)) and torch.all(kept[n:] == 9)
    check_status()


def test_grouped_neighbours_and_bad_bounds():
    from paracel_b200.ops._lib import BadDeviceId
    from paracel_b200.ops.mx4 import check_status, mx4_grouped_nt, mx4_quantize
    counts, N, K = [5, 70, 3, 130], 90, 224
    T, E = sum(counts), 4
    A, B = _grid(T, K, 1), _grid(E * N, K, 2).view(E, N, K)
    off = torch.tensor([0] + counts, device="cuda").cumsum(0)
    ref = mx4_grouped_nt(A, mx4_quantize(B), off)
    A[:5], A[75:78], B[0], B[2] = float("nan"), float("inf"), float("inf"), float("nan")
    got = mx4_grouped_nt(A, mx4_quantize(B), off)
    assert torch.equal(got[5:75], ref[5:75]) and torch.equal(got[78:], ref[78:])
    assert torch.isnan(got[:5]).all() and torch.isnan(got[75:78]).all()
    check_status()
    got = mx4_grouped_nt(A, mx4_quantize(B), torch.tensor([0, 90, 20, 1 << 35, 60], device="cuda"))
    with pytest.raises(BadDeviceId):
        check_status()
    again = mx4_grouped_nt(A, mx4_quantize(B), torch.tensor([0, 90, 90, T, T], device="cuda"))
    check_status()
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(again))


def test_tables_beyond_two_to_the_32_values():
    from paracel_b200.ops.mx4 import Mx4Matrix, mx4_dequantize, mx4_gemm_nt, mx4_quantize
    rows, K = 4_200_011, 1056
    g = torch.Generator(device="cuda").manual_seed(1)
    data = torch.randint(0, 256, (rows, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.randint(125, 130, ((K + 127) // 128, rows, 4), device="cuda", generator=g, dtype=torch.uint8)
    q = Mx4Matrix(data, scales, K)
    part = Mx4Matrix(data[-272:].contiguous(), scales[:, -272:].contiguous(), K)
    A = _grid(3, K, 2)
    got = mx4_gemm_nt(A, q, out_dtype=BF)
    assert torch.equal(got[:, -272:], mx4_gemm_nt(A, part, out_dtype=BF))
    tall = mx4_gemm_nt(q, mx4_quantize(A))
    assert torch.equal(tall[-272:], mx4_gemm_nt(part, mx4_quantize(A)))
    _near(got[:, -272:], A, mx4_dequantize(part))
    x = mx4_dequantize(q, BF)
    assert torch.equal(x[-272:], mx4_dequantize(part, BF))
    again = mx4_dequantize(mx4_quantize(x), BF)
    assert torch.equal(again[-1000:], mx4_dequantize(mx4_quantize(x[-1000:].contiguous()), BF))


def test_captured_calls_follow_their_inputs_and_streams_do_not_mix():
    from paracel_b200.ops.mx4 import check_status, mx4_gemm_nt, mx4_grouped_nt, mx4_quantize
    T, E, N, K = 300, 3, 200, 160
    A = _grid(T, K, 1)
    B = _grid(E * N, K, 2)
    q = mx4_quantize(B)
    off = torch.tensor([0, 100, 100, 300], device="cuda")
    side = torch.cuda.Stream()

    def calls():
        return mx4_gemm_nt(A, q), mx4_grouped_nt(A, q, off)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = calls()
        graphs.append((g, got))
    for seed, bounds in ((5, [0, 0, 300, 300]), (6, [0, 7, 21, 300])):
        A.copy_(_grid(T, K, seed)), off.copy_(torch.tensor(bounds))
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            eager = calls()
        torch.cuda.synchronize()
        ref = A.double() @ B.double().T
        byg = torch.cat([ref[bounds[e]:bounds[e + 1], e * N:(e + 1) * N] for e in range(E)])
        for one, two in (graphs[0][1], graphs[1][1], eager):
            assert torch.equal(one.double(), ref) and torch.equal(two.double(), byg)
    check_status()


def test_a_chain_of_calls_waits_for_what_it_reads():
    """Both operands, and the bounds, are written by the kernel right before the one that reads them, in memory that others just gave back."""
    from paracel_b200.ops.mx4 import check_status, mx4_dequantize, mx4_gemm_nt, mx4_grouped_nt, mx4_quantize
    T, E, N = 70, 3, 160
    X0, W0 = _grid(T, N, 1), _grid(E * N, N, 2)
    bounds = [torch.tensor(b, device="cuda") for b in ([0, 20, 40, 70], [0, 0, 70, 70], [0, 1, 2, 70])]

    def chain(wait):
        X, W, off, seen = X0.clone(), W0.clone(), torch.empty_like(bounds[0]), []
        for i in range(40):
            q = mx4_quantize(W)
            wait()
            off.copy_(bounds[i % 3])
            y = mx4_grouped_nt(X, q, off)
            wait()
            X = y.clamp_(-8, 8)
            z = mx4_gemm_nt(mx4_quantize(X), q)
            wait()
            X = mx4_gemm_nt(z[:, :N].contiguous(), mx4_quantize(W[:N])).clamp_(-8, 8)
            W = torch.roll(mx4_dequantize(q), i, 0)
            seen += [y, z, X.clone()]
        return seen

    apart = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), apart))
    check_status()


def test_experts_trained_in_16_bits_answer_from_four():
    """The set as it is used: rows sorted by expert, a step of training, the weights quantised, and served; each stage against the formulas."""
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_gemm_nt, mx4_grouped_nt, mx4_quantize
    T, E, H, K = 700, 5, 264, 136
    g = torch.Generator(device="cuda").manual_seed(8)
    expert = torch.randint(0, E - 1, (T,), device="cuda", generator=g).sort().values       # the last one has no row
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(expert, minlength=E).cumsum(0)
    X = torch.randn(T, K, device="cuda", generator=g).to(BF)
    W1, W2 = (torch.randn(E, *s, device="cuda", generator=g) / 12 for s in ((H, K), (K, H)))
    h = grouped_nt(X, W1.to(BF), off)
    a = h.relu()
    y = grouped_nt(a, W2.to(BF), off, out_dtype=F)
    dy = (y - X.float()).to(BF)
    da = grouped_nn(dy, W2.to(BF), off) * (h > 0)
    d1, d2 = grouped_tn(da, X, off, out_dtype=F), grouped_tn(dy, a, off, out_dtype=F)
    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        _near(d2[e], dy[r].T, a[r].T)
        _near(d1[e], da[r].T, X[r].T)
    assert not d1[-1].any() and not d2[-1].any()
    q1, q2 = mx4_quantize(W1 - 1e-3 * d1), mx4_quantize(W2 - 1e-3 * d2)
    s = mx4_grouped_nt(X, q1, off).relu()
    out = mx4_grouped_nt(s, q2, off)
    assert out.dtype == BF
    w1, w2 = mx4_dequantize(q1).view(E, H, K), mx4_dequantize(q2).view(E, K, H)
    x4, s4 = mx4_dequantize(mx4_quantize(X)), mx4_dequantize(mx4_quantize(s))
    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        if r.start < r.stop:
            ref = mx4_gemm_nt(mx4_quantize(X[r]), mx4_quantize(w1[e]), out_dtype=BF).relu()
            assert torch.equal(s[r], ref)          # the groups' products are the plain product's, row for row
            _near(out[r], s4[r], w2[e])
            _near(mx4_grouped_nt(X, q1, off, out_dtype=F)[r], x4[r], w1[e])


def test_two_threads_with_rows_of_different_lengths():
    """Few rows are quantised by the product's own blocks, whose shared memory goes with the rows' length: calls of one thread do not change what
    another's may take.  The launcher is called directly, so that the threads are in it nearly all the time."""
    import threading
    from paracel_b200.ops import _lib
    from paracel_b200.ops.mx4 import check_status, mx4_quantize
    lib, N, start, wrong, kept = _lib.load(), 1000, threading.Barrier(4, timeout=60), [], []

    def serve(i, K):
        A, B, out, stream = _grid(1, K, i), _grid(N, K, 9 + i), torch.empty(1, N, device="cuda"), torch.cuda.Stream()
        q = mx4_quantize(B)
        kept.append((A, B, q, out))
        args = (A.data_ptr(), K, 0, None, None, q.data.data_ptr(), q.scales.data_ptr(), None, 0, out.data_ptr(), N, 0, 1, 1, N, K, 1, stream.cuda_stream)
        torch.cuda.synchronize()
        start.wait()
        wrong.extend(filter(None, (lib.pcl_mx4_rows(*args) for _ in range(30000))))

    assert all(lib.pcl_mx4_room(0, 1, 1, N, K) == 0 for K in (100, 1792))         # both are of that kind
    threads = [threading.Thread(target=serve, args=a) for a in enumerate((100, 1792, 100, 1792))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    check_status()
    assert not wrong and len(kept) == 4
    for A, B, _, out in kept:
        assert torch.equal(out.double(), A.double() @ B.double().T)


def test_as_many_rows_as_a_call_takes():
    """2^31 - 513 rows against a few: quantised, multiplied by one and given back, the same values at both ends and in the middle."""
    from paracel_b200.ops.grouped import MAX_ROWS
    from paracel_b200.ops.mx4 import check_status, mx4_dequantize, mx4_gemm_nt, mx4_grouped_nt, mx4_quantize
    T, C = MAX_ROWS - 1, 8
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("not enough memory")
    X = torch.zeros(T, C, device="cuda", dtype=BF)
    windows = [slice(a, a + 3000) for a in (0, T // 2, T - 3000)]
    for i, w in enumerate(windows):
        X[w] = _grid(3000, C, i).to(BF)
    q = mx4_quantize(X)
    kept = [X[w].clone() for w in windows]
    del X
    torch.cuda.empty_cache()
    B = torch.stack((torch.eye(C, device="cuda"), 2 * torch.eye(C, device="cuda").flip(0)))
    off = torch.tensor([0, T - 1501, T], device="cuda")
    for make, factor in ((lambda: mx4_gemm_nt(q, mx4_quantize(B[0]), out_dtype=BF), None), (lambda: mx4_grouped_nt(q, mx4_quantize(B), off, out_dtype=BF), off),
                         (lambda: mx4_dequantize(q, BF), None)):
        y = make()
        check_status()
        for w, x in zip(windows, kept):
            want = x.clone()
            if factor is not None and w.stop == T:
                want[-1501:] = 2 * x[-1501:].flip(1)
            assert torch.equal(y[w], want)
        del y
    del q
    torch.cuda.empty_cache()
