"""Products grouped by expert and their gradients against plain products in 64 bits.

Tolerance of a sum of R products of 16-bit values, each exact in fp32: every one of the at most R additions is off by no more than one
unit in the last of 24 bits of a partial sum that is at most S = sum |a| |b|, so R 2^-23 S in all; then the rounding into the result's
type, half a step, eps / 2 of the value.  fp16 results below 2^-14 are 2^-24 apart.  Whole numbers whose sums stay below 2^24 come
out exactly in fp32.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _offsets(counts, first=0, dtype=torch.int32):
    return torch.tensor([first] + counts, device="cuda").cumsum(0).to(dtype)


def _bounds(offsets, T):
    out, at = [], 0
    for v in offsets.tolist():
        at = max(at, min(max(v, 0), T))
        out.append(at)
    return out


def _ref_rows(A, W, offsets):
    """(values, sums of magnitudes) of a[t] W[e]^T in 64 bits, zero for rows of no group; W [E, columns, reduction]."""
    y = torch.zeros(A.shape[0], W.shape[1], dtype=torch.float64, device=A.device)
    s = torch.zeros_like(y)
    b = _bounds(offsets, A.shape[0])
    for e in range(W.shape[0]):
        a, w = A[b[e]:b[e + 1]].double(), W[e].double()
        y[b[e]:b[e + 1]] = a @ w.T
        s[b[e]:b[e + 1]] = a.abs() @ w.abs().T
    return y, s


def _ref_tn(dY, X, offsets):
    b = _bounds(offsets, X.shape[0])
    E = len(b) - 1
    d = torch.zeros(E, dY.shape[1], X.shape[1], dtype=torch.float64, device=X.device)
    s, most = torch.zeros_like(d), 0
    for e in range(E):
        y, x = dY[b[e]:b[e + 1]].double(), X[b[e]:b[e + 1]].double()
        d[e], s[e] = y.T @ x, y.abs().T @ x.abs()
        most = max(most, b[e + 1] - b[e])
    return d, s, most


def _near(got, ref, mags, R):
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + R * 2.0 ** -23 * mags * (1 + 2.0 ** -8)
    if got.dtype == FP:
        tol += 2.0 ** -25
    off = (got.double() - ref).abs()
    assert torch.all(off <= tol), f"worst {float((off - tol).max())} beyond, at {int((off - tol).argmax())} of {off.numel()}"


def _make(T, E, N, K, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(T, K, device="cuda", generator=g).to(dtype), torch.randn(T, N, device="cuda", generator=g).to(dtype),
            torch.randn(E, N, K, device="cuda", generator=g).to(dtype))


def _whole(T, E, N, K, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randint(-4, 5, s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return f(T, K), f(T, N), f(E, N, K)


# counts, rows behind the last group, N, K
SHAPES = [
    ([1], 0, 1, 1), ([1], 0, 128, 64), ([3], 0, 8, 16), ([0, 1, 0], 0, 33, 7), ([0, 0], 5, 40, 24), ([7, 0, 9], 0, 130, 65),
    ([16, 31, 33, 1], 3, 72, 200), ([64] * 4, 0, 64, 64), ([128, 256], 0, 256, 128), ([127, 129, 255, 257], 1, 257, 129),
    ([300, 0, 0, 1, 511], 17, 520, 264), ([1000], 0, 1001, 777), ([5] * 100, 0, 100, 100), ([0] * 63 + [70], 0, 136, 328),
    ([2, 260, 3], 0, 128, 1032), ([1500, 40], 0, 384, 512), ([600, 17], 0, 900, 2050),
    # a cluster for a tile; tiles of 256 rows for one CTA, and for a pair; with ends of every kind
    ([1], 0, 300, 1000), ([3, 0, 1], 2, 256, 520), ([33, 64], 0, 130, 4100), ([700, 0, 1300, 33, 256], 5, 2000, 1900),
    ([700, 0, 1300, 33, 256], 5, 4008, 3800), ([257, 15, 1000, 0, 500, 470, 60], 0, 3777, 4001),
    # tn by pairs with columns in whole blocks of 64, an odd number of them
    ([30, 0, 65, 64, 1] * 20, 0, 320, 256), ([200, 7] * 40, 3, 64, 640), ([63, 65, 128, 0] * 16, 0, 448, 320),
    # tn by clusters: groups without rows for some of the CTAs, or for any; ends of every kind; 64 columns and 128
    ([1500, 0, 3, 70], 9, 96, 200), ([2000], 0, 1, 9), ([0, 4000, 65], 0, 72, 520), ([3000, 5000, 129], 2, 200, 328),
    ([9001], 1, 777, 1030), ([8192, 0], 0, 512, 512), ([700, 1400, 0, 31], 0, 1144, 128), ([20000], 0, 67, 65),
]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("counts,spare,N,K", SHAPES)
def test_grouped_products_match(counts, spare, N, K, dtype):
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    T, E = sum(counts) + spare, len(counts)
    X, dY, W = _make(T, E, N, K, dtype)
    off = _offsets(counts)
    for out_dtype in (dtype, torch.float32):
        y = grouped_nt(X, W, off, out_dtype=out_dtype)
        z = grouped_nn(dY, W, off, out_dtype=out_dtype)
        d = grouped_tn(dY, X, off, out_dtype=out_dtype)
        check_status()
        _near(y, *_ref_rows(X, W, off), K)
        _near(z, *_ref_rows(dY, W.transpose(1, 2), off), N)
        ref, mags, most = _ref_tn(dY, X, off)
        _near(d, ref, mags, most)
        b = _bounds(off, T)
        assert not y[b[-1]:].any() and not z[b[-1]:].any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("counts,spare,N,K", SHAPES)
def test_grouped_products_of_whole_numbers_are_exact(counts, spare, N, K, dtype):
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    T, E = sum(counts) + spare, len(counts)
    X, dY, W = _whole(T, E, N, K, dtype)
    off = _offsets(counts, dtype=torch.int64)
    f = torch.float32
    assert torch.equal(grouped_nt(X, W, off, out_dtype=f).double(), _ref_rows(X, W, off)[0])
    assert torch.equal(grouped_nn(dY, W, off, out_dtype=f).double(), _ref_rows(dY, W.transpose(1, 2), off)[0])
    assert torch.equal(grouped_tn(dY, X, off, out_dtype=f).double(), _ref_tn(dY, X, off)[0])


@pytest.mark.parametrize("first,spare", [(0, 9), (4, 0), (37, 30)])
def test_rows_of_no_group_stay_as_they_were(first, spare):
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt
    counts, N, K = [20, 0, 150], 72, 40
    T = first + sum(counts) + spare
    X, dY, W = _whole(T, 3, N, K, BF)
    # what rows of no group hold reaches nothing
    X[:first], X[first + 170:], dY[:first], dY[first + 170:] = float("nan"), float("inf"), float("inf"), float("nan")
    off = _offsets(counts, first)
    for call, A, M in ((grouped_nt, X, W), (grouped_nn, dY, W)):
        ref = _ref_rows(A, M if call is grouped_nt else M.transpose(1, 2), off)[0]
        wide = torch.full((T, ref.shape[1] + 11), -7.0, device="cuda")
        call(A, M, off, out=wide[:, 3:-8])
        want = wide.new_full(wide.shape, -7.0).double()
        want[first:first + 170, 3:-8] = ref[first:first + 170]
        assert torch.equal(wide.double(), want)
        assert torch.equal(call(A, M, off, out_dtype=torch.float32).double(), ref)


def test_what_one_group_holds_does_not_reach_another():
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    counts, N, K = [5, 70, 3, 130, 1], 90, 200
    T = sum(counts)
    X, dY, W = _whole(T, 5, N, K, FP)
    off = _offsets(counts)
    b = off.tolist()
    bad = [0, 2, 4]
    X2, dY2, W2 = X.clone(), dY.clone(), W.clone()
    for e in bad:
        X2[b[e]:b[e + 1]], dY2[b[e]:b[e + 1]], W2[e] = float("nan"), float("inf"), float("nan")
    y, z, d = grouped_nt(X2, W2, off), grouped_nn(dY2, W2, off), grouped_tn(dY2, X2, off)
    ry, rz, rd = grouped_nt(X, W, off), grouped_nn(dY, W, off), grouped_tn(dY, X, off)
    for e in (1, 3):
        assert torch.equal(y[b[e]:b[e + 1]], ry[b[e]:b[e + 1]])
        assert torch.equal(z[b[e]:b[e + 1]], rz[b[e]:b[e + 1]])
        assert torch.equal(d[e], rd[e])
    for e in bad:
        assert not torch.isfinite(y[b[e]:b[e + 1]]).any() and not torch.isfinite(z[b[e]:b[e + 1]]).any()
        assert not torch.isfinite(d[e]).any()


def test_infinities_stay_in_their_place():
    from paracel_b200.ops.grouped import grouped_nt, grouped_tn
    X, dY, W = (t.abs() + 1 for t in _whole(200, 2, 64, 96, BF))
    off = _offsets([90, 110])
    X[17, 5], W[1, 3, 7] = float("inf"), float("nan")
    y, ref = grouped_nt(X, W, off, out_dtype=torch.float32).double(), _ref_rows(X, W, off)[0]
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(torch.isinf(y), torch.isinf(ref))
    d, ref = grouped_tn(dY, X, off, out_dtype=torch.float32).double(), _ref_tn(dY, X, off)[0]
    assert torch.equal(d, ref)


@pytest.mark.parametrize("raw,T", [([0, 50, 20, 90], 90), ([-5, 30, 30, 200], 90), ([60, 10, 10, 10], 90),
                                   ([0, 1 << 40, 5, -(1 << 40)], 90)])
def test_bad_bounds_are_moved_and_reported(raw, T):
    from paracel_b200.ops._lib import BadDeviceId
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    X, dY, W = _whole(T, 3, 40, 24, BF)
    off = torch.tensor(raw, device="cuda")
    f = torch.float32
    for call, got in ((grouped_nt, lambda: _ref_rows(X, W, off)[0]), (grouped_nn, lambda: _ref_rows(dY, W.transpose(1, 2), off)[0])):
        y = call(X if call is grouped_nt else dY, W, off, out_dtype=f)
        with pytest.raises(BadDeviceId):
            check_status()
        assert torch.equal(y.double(), got())
        check_status()                                  # reported once
    d = grouped_tn(dY, X, off, out_dtype=f)
    with pytest.raises(BadDeviceId):
        check_status(X.device)
    assert torch.equal(d.double(), _ref_tn(dY, X, off)[0])


def test_strided_operands_and_results():
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    counts, N, K = [33, 100, 7], 104, 80
    T, E = sum(counts), 3
    off = _offsets(counts)
    big, bigy, bigw = _whole(T, E, N, 2 * K, BF)[0], _whole(T, E, 3 * N, K, BF)[1], _whole(T, 2 * E, N + 8, K + 16, BF)[2]
    f = torch.float32
    variants = [
        (big[:, :K], bigy[:, N:2 * N], bigw[::2, :N, 8:K + 8]),          # rows at multiples of 16 bytes: read where they lie
        (big[:, 1:K + 1], bigy[:, 3:N + 3], bigw[:E, 5:N + 5, 1:K + 1]),  # copied
        (big[:, ::2], bigy[:, ::3], bigw[:E, :K].transpose(1, 2)[:, :K, :K]),
        (big[:1, :K].expand(T, K), bigy[:1, :N].expand(T, N), bigw[:1, :N, :K].expand(E, N, K)),
    ]
    for X, dY, W in variants:
        if W.shape[1] != N:
            dY = dY[:, :W.shape[1]]
        assert torch.equal(grouped_nt(X, W, off, out_dtype=f).double(), _ref_rows(X, W, off)[0])
        assert torch.equal(grouped_nn(dY, W, off, out_dtype=f).double(), _ref_rows(dY, W.transpose(1, 2), off)[0])
        assert torch.equal(grouped_tn(dY, X, off, out_dtype=f).double(), _ref_tn(dY, X, off)[0])
    X, dY, W = variants[0]
    # results at every offset of a line, two and four bytes a value
    for dtype in (BF, f):
        for shift in (0, 1, 2, 4, 8):
            wide = torch.full((T, N + 32), 5.0, device="cuda", dtype=dtype)
            grouped_nt(X, W, off, out=wide[:, shift:shift + N])
            ref = torch.full_like(wide, 5.0)
            ref[:, shift:shift + N] = grouped_nt(X, W, off, out_dtype=dtype)
            assert torch.equal(wide, ref)
    flat = torch.full((E * N * K + 3,), 5.0, device="cuda", dtype=BF)
    grouped_tn(dY, X, off, out=flat[1:-2].view(E, N, K))
    assert torch.equal(flat[1:-2].view(E, N, K), grouped_tn(dY, X, off))
    assert flat[0] == 5 and torch.all(flat[-2:] == 5)


def test_gradients_match_differences():
    """The product is linear in either operand: with whole numbers its differences are exact."""
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    counts, N, K = [20, 1, 0, 77], 48, 56
    T, E = sum(counts), 4
    off = _offsets(counts)
    X, dY, W = _whole(T, E, N, K, BF)
    hX, _, hW = _whole(T, E, N, K, BF, seed=9)
    f = torch.float32
    loss = lambda x, w: (grouped_nt(x, w, off, out_dtype=f).double() * dY.double()).sum()  # noqa: E731
    dx, dw = grouped_nn(dY, W, off, out_dtype=f), grouped_tn(dY, X, off, out_dtype=f)
    assert loss(X + hX, W) - loss(X, W) == (dx.double() * hX.double()).sum()
    assert loss(X, W + hW) - loss(X, W) == (dw.double() * hW.double()).sum()


def test_empty_calls():
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    X, dY, W = _whole(0, 2, 24, 16, BF)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert grouped_nt(X, W, off).shape == (0, 24) and grouped_nn(dY, W, off).shape == (0, 16)
    assert torch.equal(grouped_tn(dY, X, off), torch.zeros(2, 24, 16, device="cuda", dtype=BF))


def test_largest_group_count_and_ties_with_one_group():
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 5, (1024,), generator=g).tolist()
    T = sum(counts)
    X, dY, W = _whole(T, 1024, 24, 32, FP)
    off, f = _offsets(counts), torch.float32
    assert torch.equal(grouped_nt(X, W, off, out_dtype=f).double(), _ref_rows(X, W, off)[0])
    assert torch.equal(grouped_nn(dY, W, off, out_dtype=f).double(), _ref_rows(dY, W.transpose(1, 2), off)[0])
    assert torch.equal(grouped_tn(dY, X, off, out_dtype=f).double(), _ref_tn(dY, X, off)[0])


@pytest.mark.parametrize("N,K", [(72, 1056), (1056, 72)])
def test_operands_beyond_two_to_the_31_values(N, K):
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    T = 2_100_007
    g = torch.Generator(device="cuda").manual_seed(4)
    X = torch.randint(-2, 3, (T, K), device="cuda", generator=g, dtype=torch.int8).to(BF)
    W = torch.randint(-2, 3, (3, N, K), device="cuda", generator=g).to(BF)
    off = torch.tensor([0, 100, T - 300, T], device="cuda")
    tail = slice(T - 300, T)
    local = torch.tensor([0, 300], device="cuda")
    y = grouped_nt(X, W, off)
    assert torch.equal(y[tail].double(), _ref_rows(X[tail], W[2:], local)[0].to(BF).double())
    z = grouped_nn(y, W, off)
    ref, mags = _ref_rows(y[tail], W[2:].transpose(1, 2), local)
    _near(z[tail], ref, mags, N)
    d = grouped_tn(y, X, off, out_dtype=torch.float32)
    ref, mags, most = _ref_tn(y[tail], X[tail], local)
    _near(d[2:], ref, mags, most)


def test_a_captured_step_follows_its_inputs():
    """Forward and both gradients in one graph; bounds, rows and matrices change between replays.  A second graph and an
    eager call run in between on another stream."""
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    T, E, N, K = 400, 6, 136, 96
    X, dY, W = _whole(T, E, N, K, BF)
    off = _offsets([100, 50, 0, 150, 60, 40])
    f = torch.float32

    def step():
        return (grouped_nt(X, W, off, out_dtype=f), grouped_nn(dY, W, off, out_dtype=f), grouped_tn(dY, X, off, out_dtype=f))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    for seed, counts in ((5, [0, 0, 400, 0, 0, 0]), (6, [1, 2, 3, 4, 5, 6]), (7, [200, 0, 0, 0, 0, 200])):
        x, y, w = _whole(T, E, N, K, BF, seed)
        X.copy_(x), dY.copy_(y), W.copy_(w), off.copy_(_offsets(counts))
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            eager = step()
        torch.cuda.synchronize()
        ref = (_ref_rows(X, W, off)[0], _ref_rows(dY, W.transpose(1, 2), off)[0], _ref_tn(dY, X, off)[0])
        for got in (graphs[0][1], graphs[1][1], eager):
            for a, b in zip(got, ref):
                assert torch.equal(a.double(), b)
    check_status()


def test_calls_on_two_streams_at_once():
    from paracel_b200.ops.grouped import grouped_nt, grouped_tn
    T, E, N, K = 3000, 8, 520, 512
    X, dY, W = _whole(T, E, N, K, BF)
    off = _offsets([375] * 8)
    ref, rd = _ref_rows(X, W, off)[0], _ref_tn(dY, X, off)[0]
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append((grouped_nt(X, W, off, out_dtype=torch.float32), grouped_tn(dY, X, off, out_dtype=torch.float32)))
    torch.cuda.synchronize()
    for y, d in got:
        assert torch.equal(y.double(), ref) and torch.equal(d.double(), rd)


def test_a_chain_of_calls_waits_for_what_it_reads():
    """Every call reads what the one right before it wrote, operands and bounds among it, and takes over memory that others just gave back: kernels
    that begin before their predecessor has ended must not be seen to."""
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    T, E, N, K = 96, 4, 136, 72
    X0, _, W0 = _whole(T, E, N, K, BF, seed=3)
    bounds = [_offsets(c) for c in ([24, 24, 24, 24], [0, 90, 1, 5], [96, 0, 0, 0], [3, 3, 3, 80])]

    def chain(wait):
        off, X, W, seen = torch.empty_like(bounds[0]), X0.clone(), W0.clone(), []
        for i in range(60):
            off.copy_(bounds[i % 4])
            y = grouped_nt(X, W, off)
            wait()
            y.clamp_(-8, 8)
            z = grouped_nn(y, W, off)
            wait()
            X = z.clamp_(-4, 4)
            d = grouped_tn(y, X, off)
            wait()
            W = d.clamp_(-4, 4)
            a = grouped_nt(X, W, off)
            b = grouped_nt(X, W, off, out=torch.empty_like(a))
            wait()
            W = grouped_tn(a, X, off).clamp_(-4, 4)
            seen += [a.clone(), b, W]
        return seen

    apart = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), apart))
    check_status()


def test_a_reduction_over_a_million_rows():
    from paracel_b200.ops.grouped import check_status, grouped_tn
    T, N, K = 1_000_003, 40, 72
    g = torch.Generator(device="cuda").manual_seed(6)
    X = torch.randint(-1, 2, (T, K), device="cuda", generator=g, dtype=torch.int8)
    dY = torch.randint(-1, 2, (T, N), device="cuda", generator=g, dtype=torch.int8)
    off = torch.tensor([0, T - 3, T], device="cuda")
    d = grouped_tn(dY.to(FP), X.to(FP), off, out_dtype=torch.float32)
    check_status()
    assert torch.equal(d[0].double(), dY[:-3].double().T @ X[:-3].double())
    assert torch.equal(d[1].double(), dY[-3:].double().T @ X[-3:].double())


def test_the_same_call_gives_the_same_bits():
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    X, dY, W = _make(2000, 5, 264, 1032, BF)
    off = _offsets([1, 999, 0, 500, 500])
    first = (grouped_nt(X, W, off), grouped_nn(dY, W, off), grouped_tn(dY, X, off))
    for _ in range(3):
        again = (grouped_nt(X, W, off), grouped_nn(dY, W, off), grouped_tn(dY, X, off))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_training_steps_of_a_grouped_layer():
    """Rows sorted by cluster, a matrix for each, squared error: every step is what the formulas give from the same weights."""
    from paracel_b200.ops.grouped import check_status, grouped_nt, grouped_tn
    T, E, N, K = 900, 4, 40, 56
    g = torch.Generator(device="cuda").manual_seed(2)
    cluster = torch.randint(0, E, (T,), device="cuda", generator=g)
    order = cluster.argsort()
    off = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    off[1:] = torch.bincount(cluster, minlength=E).cumsum(0)
    X = torch.randn(T, K, device="cuda", generator=g).to(BF)[order]
    target = torch.randn(T, N, device="cuda", generator=g)
    W = torch.randn(E, N, K, device="cuda", generator=g) / 8
    for _ in range(3):
        Wh = W.to(BF)
        y = grouped_nt(X, Wh, off, out_dtype=torch.float32)
        _near(y, *_ref_rows(X, Wh, off), K)
        dY = ((y - target) / T).to(BF)
        dW = grouped_tn(dY, X, off, out_dtype=torch.float32)
        ref, mags, most = _ref_tn(dY, X, off)
        _near(dW, ref, mags, most)
        W -= 0.5 * dW
    check_status()


@pytest.mark.parametrize("mats,rows,cols,step,extra,start", [
    (1, 1, 1, 1, 0, 1), (1, 5, 7, 7, 0, 0), (1, 3, 8, 9, 0, 0), (2, 4, 9, 10, 3, 1), (3, 33, 20, 22, 0, 2), (1, 300, 33, 36, 0, 4), (2, 9, 1000, 1001, 1, 3),
    (1, 3, 1031, 1032, 0, 5), (5, 1, 2050, 2051, 0, 0), (1, 2, 9001, 9001, 0, 7), (4, 17, 64, 0, 40, 1), (1, 70000, 3, 3, 0, 0), (1025, 2, 13, 13, 0, 3),
])
def test_operands_are_copied_to_whole_rows(mats, rows, cols, step, extra, start):
    """Copies of the exact bits, of one operand and of two, zeros behind each row's end and nothing written outside."""
    from paracel_b200.ops import _lib
    step_e = rows * step + extra
    need = start + (mats - 1) * step_e + (rows - 1) * step + cols
    pitch = (cols + 7) // 8 * 8
    flat = torch.randint(-32768, 32767, (need,), dtype=torch.int16, device="cuda")
    src = flat.as_strided((mats, rows, cols), (step_e, step, 1), start)
    other = torch.randint(-32768, 32767, (19, 5), dtype=torch.int16, device="cuda")
    second = torch.full((19, 8), 77, dtype=torch.int16, device="cuda")
    for both in (False, True):
        room = torch.full((8 + mats * rows * pitch + 8,), 77, dtype=torch.int16, device="cuda")
        dst = room[8:-8].view(mats, rows, pitch)
        tail = (other.data_ptr(), 95, 5, 1, 19, 5, second.data_ptr(), 0, 0) if both else (0,) * 9
        _lib.call_on(0, "pcl_grouped_pad", src.data_ptr(), step_e, step, mats, rows, cols, dst.data_ptr(), *tail)
        assert torch.equal(dst[..., :cols], src) and not dst[..., cols:].any()
        assert bool((room[:8] == 77).all()) and bool((room[-8:] == 77).all())
        assert torch.equal(second[:, :5], other) == both and bool((second[:, 5:] == (0 if both else 77)).all())


@pytest.mark.parametrize("N,K,left", [(64, 128, 0), (200, 132, 1), (72, 260, 4), (130, 96, 8), (16, 33, 0), (256, 512, 3)])
def test_results_of_32_bits_in_strided_rows(N, K, left):
    """Rows at multiples of 16 bytes and elsewhere, m that ends inside a store, column counts that are no multiple of 16."""
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt
    counts = [17, 0, 70, 300, 1]
    T = sum(counts)
    X, dY, W = _whole(T, 5, N, K, BF)
    off = _offsets(counts)
    for call, A, M, cols in ((grouped_nt, X, W, N), (grouped_nn, dY, W.transpose(1, 2), K)):
        for room in (left + cols, left + cols + 4, left + (cols + 7) // 4 * 4):
            wide = torch.full((T, room), 5.0, device="cuda")
            call(A, W, off, out=wide[:, left:left + cols])
            ref = torch.full((T, room), 5.0, device="cuda", dtype=torch.float64)
            ref[:, left:left + cols] = _ref_rows(A, M, off)[0]
            assert torch.equal(wide.double(), ref)


@pytest.mark.parametrize("bounds,dtype", [([0, 0, 3, 3, 40], torch.int32), ([5, 4, 9, 9, 2], torch.int64), ([0, 1, 2, 3, 4], torch.int64), ([7, 7, 7, 7, 7], torch.int32),
                                          ([-3, 2, -1, 50, 60], torch.int32)])
def test_only_matrices_of_groups_with_rows_are_copied(bounds, dtype):
    """What a call does not copy it does not read: the memory of a copy is whatever was there before."""
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt
    N, K, T = 45, 37, 40
    X, dY, W = _whole(T, 4, N, K, BF)
    off = torch.tensor(bounds, dtype=dtype, device="cuda")
    fixed, top = [], 0
    for v in bounds:
        top = max(top, min(max(v, 0), T))
        fixed.append(top)
    good = torch.tensor(fixed, dtype=dtype, device="cuda")
    f = torch.float32
    for _ in range(3):
        spoiled = [torch.full((4 * N * 48,), float("nan"), dtype=BF, device="cuda") for _ in range(4)]
        del spoiled
        assert torch.equal(grouped_nt(X, W, off, out_dtype=f).double(), _ref_rows(X, W, good)[0])
        assert torch.equal(grouped_nn(dY, W, off, out_dtype=f).double(), _ref_rows(dY, W.transpose(1, 2), good)[0])
    try:
        check_status()
    except Exception:
        assert bounds != fixed


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("E,N,K,shift", [(3, 1, 1, 0), (40, 300, 7, 1), (9, 257, 129, 3), (600, 256, 640, 2), (300, 513, 258, 5), (5, 64, 1000, 0)])
def test_gradients_of_groups_without_rows_are_zero(E, N, K, shift, dtype):
    """Every value of the result is written, and none outside, wherever it begins."""
    from paracel_b200.ops.grouped import grouped_tn
    counts = [0] * E
    counts[E // 2] = 5
    X, dY, _ = _whole(5, 1, N, K, BF)
    off = _offsets(counts)
    flat = torch.full((E * N * K + 16,), 7.0, device="cuda", dtype=dtype)
    out = flat[shift:shift + E * N * K].view(E, N, K)
    grouped_tn(dY, X, off, out=out)
    assert torch.equal(out.double(), _ref_tn(dY, X, off)[0].to(dtype).double())
    assert bool((flat[:shift] == 7).all()) and bool((flat[shift + E * N * K:] == 7).all())


def test_odd_widths_into_given_results_on_a_stream_and_in_a_graph():
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    counts, N, K = [33, 0, 100, 7], 45, 77
    T, E = sum(counts), 4
    X, dY, W = _whole(T, E, N, K, BF)
    off = _offsets(counts)
    f = torch.float32
    y, z, d = torch.empty(T, N, device="cuda"), torch.empty(T, K, device="cuda"), torch.empty(E, N, K, device="cuda")

    def calls():
        grouped_nt(X, W, off, out=y)
        grouped_nn(dY, W, off, out=z)
        grouped_tn(dY, X, off, out=d)
        return grouped_nt(X, W, off, out_dtype=f), grouped_nn(dY, W, off, out_dtype=f), grouped_tn(dY, X, off, out_dtype=f)

    def right(made):
        for got, want in ((y, _ref_rows(X, W, off)[0]), (z, _ref_rows(dY, W.transpose(1, 2), off)[0]), (d, _ref_tn(dY, X, off)[0])):
            assert torch.equal(got.double(), want)
        for got, same in zip(made, (y, z, d)):
            assert torch.equal(got, same)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        made = calls()
    torch.cuda.current_stream().wait_stream(side)
    right(made)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = calls()
    for seed in (2, 3):
        for t, new in zip((X, dY, W), _whole(T, E, N, K, BF, seed=seed)):
            t.copy_(new)
        off.copy_(_offsets([7, 100, 0, 33] if seed == 2 else [0, 0, 140, 0]))
        graph.replay()
        right(made)


@pytest.mark.parametrize("E,N,K", [(5, 1, 64), (9, 1, 33), (1, 7, 24), (6, 5, 1), (4, 1, 1)])
def test_matrices_and_rows_with_a_dimension_of_one(E, N, K):
    """Such a dimension may report any stride: it is not looked at."""
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt, grouped_tn
    T = 3 * E
    X, dY, flat = _whole(T, 1, N, K, BF)[0], _whole(T, 1, N, K, BF)[1], _whole(1, max(E, N) * E, N, K, BF)[2].view(-1)
    W = flat.as_strided((E, N, K), (N * K, K if N > 1 else K * E, 1 if K > 1 else 7))
    one = X.as_strided((1, K), (5, 1))
    off, f = _offsets([3] * E), torch.float32
    y, z, d = (torch.empty(s, device="cuda") for s in ((T, N), (T, K), (E, N, K)))
    grouped_nt(X, W, off, out=y), grouped_nn(dY, W, off, out=z), grouped_tn(dY, X, off, out=d)
    for got, given, ref in ((grouped_nt(X, W, off, out_dtype=f), y, _ref_rows(X, W, off)[0]),
                            (grouped_nn(dY, W, off, out_dtype=f), z, _ref_rows(dY, W.transpose(1, 2), off)[0]),
                            (grouped_tn(dY, X, off, out_dtype=f), d, _ref_tn(dY, X, off)[0])):
        assert torch.equal(got.double(), ref) and torch.equal(given, got)
    assert torch.equal(grouped_nt(one, W, _offsets([1] + [0] * (E - 1)), out_dtype=f).double(), X[:1].double() @ W[0].double().T)


def test_a_tail_behind_seconds_of_other_tiles():
    """A group of whole stages takes some 2.5 s before the first tile of a group with an odd number of rows: the warp that waits for such an end passes over
    the tiles without one at once, and its limit (2 s, and 2 us a stage) counts theirs.  Rows that overlap (8 values apart) keep the operands small; sums
    of -1, 0 and 1 over 7.3 million rows are exact in fp32."""
    from paracel_b200.ops.grouped import check_status, grouped_tn
    first, last, N, K = 64 * 114688, 37, 16384, 16384
    T = first + last
    g = torch.Generator(device="cuda").manual_seed(5)
    X, dY = (torch.randint(-1, 2, (8 * T + K,), device="cuda", generator=g, dtype=torch.int8).to(BF).as_strided((T, K), (8, 1)) for _ in range(2))
    off = torch.tensor([0, first, T], device="cuda")
    d = grouped_tn(dY, X, off, out_dtype=torch.float32)
    check_status()
    n, k = (torch.randint(0, K, (12,), device="cuda", generator=g) for _ in range(2))
    assert torch.equal(d[0][n][:, k].double(), dY[:first, n].double().T @ X[:first, k].double())
    assert torch.equal(d[1].double(), dY[first:].double().T @ X[first:].double())


@pytest.mark.parametrize("four_bits", [False, True])
def test_a_report_is_taken_whole_and_once(four_bits):
    """Three threads ask on streams of their own while calls report one at a time: every report reaches one of them, and none two."""
    import threading
    import time
    from paracel_b200.ops import grouped, mx4
    from paracel_b200.ops._lib import BadDeviceId
    X, W, off = torch.ones(2, 16, device="cuda", dtype=BF), torch.ones(1, 16, 16, device="cuda", dtype=BF), torch.tensor([0, 5], device="cuda")
    q = mx4.mx4_quantize(W)
    call, check = ((lambda: mx4.mx4_grouped_nt(X, q, off)), mx4.check_status) if four_bits else ((lambda: grouped.grouped_nt(X, W, off)), grouped.check_status)
    raised, odd, stop = [], [], threading.Event()

    def ask():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while not stop.is_set():
                    try:
                        check()
                    except BadDeviceId as e:
                        raised.append((e.position, e.bad_id))
        except Exception as e:
            odd.append(e)

    threads = [threading.Thread(target=ask) for _ in range(3)]
    for t in threads:
        t.start()
    try:
        for n in range(1, 201):
            call()                                       # one block, in which one thread meets the bound
            torch.cuda.current_stream().synchronize()
            until = time.monotonic() + 20
            while len(raised) < n and not odd and time.monotonic() < until:
                time.sleep(0.0005)
            time.sleep(0.002)                            # room for another to have it too
    finally:
        stop.set()
        for t in threads:
            t.join()
    assert not odd and raised == [(1, 5)] * 200
    check()


@pytest.mark.parametrize("cols", [1, 3, 7, 8, 9, 15, 19, 30, 31, 33, 37, 130, 291, 1999])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_columns_beside_a_given_result_stay(cols, dtype):
    """Rows at multiples of 16 bytes whose length is none: nothing is written behind a row's last value, nor before its first."""
    from paracel_b200.ops.grouped import grouped_nn, grouped_nt
    from paracel_b200.ops.mx4 import mx4_dequantize, mx4_gemm_nt, mx4_grouped_nt, mx4_quantize
    R = 24
    for counts in ([70, 0, 33], [5, 0, 64], [1500, 600, 700]):
        T, E = sum(counts) + 3, len(counts)
        X, _, W = _whole(T, E, cols, R, dtype)
        off, q = _offsets(counts), mx4_quantize(W)
        ref, n = _ref_rows(X, W, off)[0], T - 3
        x4 = mx4_dequantize(mx4_quantize(X)).double()
        ref4 = torch.cat([x4[a:b] @ mx4_dequantize(q)[e * cols:(e + 1) * cols].double().T for e, (a, b) in enumerate(zip(off.tolist(), off.tolist()[1:]))])
        calls = [(lambda o: grouped_nt(X, W, off, out=o), ref), (lambda o: grouped_nn(X, W.transpose(1, 2).contiguous(), off, out=o), ref),
                 (lambda o: mx4_grouped_nt(X, q, off, out=o), ref4), (lambda o: mx4_gemm_nt(X[:n], mx4_quantize(W[0]), out=o[:n]), x4[:n] @ mx4_dequantize(q)[:cols].double().T)]
        for before, behind in ((0, 0), (0, 8), (8, 0), (8, 16)):
            for call, want in calls:
                wide = torch.full((T, before + (cols + 7) // 8 * 8 + behind), -7.0, device="cuda", dtype=dtype)
                call(wide[:, before:before + cols])
                full = torch.full_like(wide, -7.0)
                full[:n, before:before + cols] = want[:n]
                assert torch.equal(wide, full)


def test_as_many_rows_as_a_call_takes():
    """2^31 - 513 rows, nearly all of one group, its bounds included; rows are zero but for three windows, and whole numbers."""
    from paracel_b200.ops.grouped import MAX_ROWS, check_status, grouped_nn, grouped_nt, grouped_tn
    T, C = MAX_ROWS - 1, 8
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("not enough memory")
    g = torch.Generator(device="cuda").manual_seed(1)
    bounds = [0, 100, T - 1501, T]
    off = torch.tensor(bounds, device="cuda")
    X, W = torch.zeros(T, C, device="cuda", dtype=BF), torch.randint(-3, 4, (3, C, C), device="cuda", generator=g).to(BF)
    windows = [(a, a + 3000) for a in (0, T // 2, T - 3000)]
    for a, b in windows:
        X[a:b] = torch.randint(-3, 4, (b - a, C), device="cuda", generator=g).to(BF)
    parts = [(max(a, lo), min(b, hi), e) for a, b in windows for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])) if max(a, lo) < min(b, hi)]
    for call, M in ((grouped_nt, W.transpose(1, 2)), (grouped_nn, W)):
        y = call(X, W, off)
        check_status()
        for a, b, e in parts:
            assert torch.equal(y[a:b].double(), X[a:b].double() @ M[e].double())
        del y
    d = grouped_tn(X, X, off, out_dtype=torch.float32)
    check_status()
    want = torch.zeros(3, C, C, device="cuda", dtype=torch.float64)
    for a, b, e in parts:
        want[e] += X[a:b].double().T @ X[a:b].double()
    assert torch.equal(d.double(), want)
    del X
    torch.cuda.empty_cache()


def _one_sign(shape, g):
    return torch.rand(shape, device="cuda", generator=g).to(BF)


@pytest.mark.parametrize("T,N,K,which", [(6000, 512, 300_001, "nt"), (300, 64, 1_000_000, "nt"), (6000, 262_144, 512, "nn"), (262_144, 2560, 2560, "tn"),
                                         (262_144, 4096, 4096, "tn"), (1_000_003, 200, 264, "tn"), (3_000_000, 128, 64, "tn")])
def test_the_error_of_long_sums_does_not_grow(T, N, K, which):
    """Sums of hundreds of thousands of terms of one sign, the worst case of additions that cut off: a part of at most 8192 terms is off by 8192 2^-23 of its own
    sum, as at the head of this file, and adding P parts up by P 2^-24 of the whole, rounded."""
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    g = torch.Generator(device="cuda").manual_seed(7)
    f = torch.float32
    if which == "tn":
        X, dY, off = _one_sign((T, K), g), _one_sign((T, N), g), torch.tensor([0, T], device="cuda")
        got, R = grouped_tn(dY, X, off, out_dtype=f)[0][:64, :64], T
        ref = dY[:, :64].double().T @ X[:, :64].double()
    else:
        A, W, off = _one_sign((T, K if which == "nt" else N), g), _one_sign((1, N, K), g), torch.tensor([0, T], device="cuda")
        got, R = (grouped_nt if which == "nt" else grouped_nn)(A, W, off, out_dtype=f)[-64:, :64], A.shape[1]
        M = W[0, :64].T if which == "nt" else W[0, :, :64]
        ref = A[-64:].double() @ M.double()
    check_status()
    parts = -(-R // 8192) + 8                            # and a last one for each of eight CTAs
    worst = float(((got.double() - ref).abs() / ref).max())
    assert worst <= 8192 * 2.0 ** -23 + parts * 2.0 ** -24, worst


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("counts,N,K", [([8192], 64, 8192), ([8193, 0, 8256], 72, 8257), ([40_000, 3, 0, 9000], 136, 20_000), ([9000] * 4, 8200, 264),
                                        ([8200] * 9, 1000, 16_448), ([140_000], 1030, 520), ([100, 30_000, 64 * 129], 520, 1048),
                                        # pairs of CTAs with several tiles each: short, long, long, short, empty
                                        ([64, 9000, 20_000, 100, 0, 8300, 5, 5, 16_385] * 2, 1536, 1280), ([9000, 17, 200, 8300] * 9, 1030, 1001)])
def test_long_reductions_of_whole_numbers_are_exact(counts, N, K, dtype):
    """Reductions in several parts and in one next to each other, in every direction and shape of tiles."""
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    T, E = sum(counts), len(counts)
    X, dY, W = _whole(T, E, N, K, dtype)
    off, f = _offsets(counts), torch.float32
    for od in (f, dtype):
        y, z, d = grouped_nt(X, W, off, out_dtype=od), grouped_nn(dY, W, off, out_dtype=od), grouped_tn(dY, X, off, out_dtype=od)
        check_status()
        assert torch.equal(y, _ref_rows(X, W, off)[0].to(f).to(od))
        assert torch.equal(z, _ref_rows(dY, W.transpose(1, 2), off)[0].to(f).to(od))
        assert torch.equal(d, _ref_tn(dY, X, off)[0].to(f).to(od))


@pytest.mark.parametrize("bounds", [[0, 0, 3, 3, 40], [5, 4, 9, 9, 2], [0, 1, 2, 3, 4], [7, 7, 7, 7, 7], [-3, 2, -1, 50, 60]])
@pytest.mark.parametrize("N,K", [(45, 37), (48, 40)])
def test_moved_bounds_and_no_others_are_reported_as_such(bounds, N, K):
    """By every product, with operands that are copied first and with others: the place and the number of a bound that had to be moved."""
    from paracel_b200.ops import mx4
    from paracel_b200.ops._lib import BadDeviceId
    from paracel_b200.ops.grouped import check_status, grouped_nn, grouped_nt, grouped_tn
    T = 40
    X, dY, W = _whole(T, 4, N, K, BF)
    off, q = torch.tensor(bounds, device="cuda"), mx4.mx4_quantize(W)
    moved, top = {}, 0
    for i, v in enumerate(bounds):
        top = max(top, min(max(v, 0), T))
        if v != top:
            moved[i] = {v, min(max(v, 0), T)}            # as given, or as cut to the rows before it is made ascending
    for call, check in ((lambda: grouped_nt(X, W, off), check_status), (lambda: grouped_nn(dY, W, off), check_status), (lambda: grouped_tn(dY, X, off), check_status),
                        (lambda: mx4.mx4_grouped_nt(X, q, off), mx4.check_status)):
        check()
        call()
        if moved:
            with pytest.raises(BadDeviceId) as e:
                check()
            assert e.value.position in moved and e.value.bad_id in moved[e.value.position]
        check()
