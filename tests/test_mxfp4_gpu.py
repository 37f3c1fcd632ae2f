"""Microscaled 4-bit matrices on the GPU against the 64-bit oracle: quantisation bit for bit, values, products."""
import numpy as np
import pytest
import torch

from aiehlc_b200.ops import Context, MxFp4
from oracle import mxfp4 as X

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _matrix(rows, cols, seed, spread=3.0):
    """Normal values whose rows and blocks differ in size by powers of two."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-spread, spread + 1, (rows, 1)))
    return torch.from_numpy(x * np.exp2(rng.integers(-spread, spread + 1, (1, X.blocks(cols))).repeat(32, 1)[:, :cols]))


def _to_gpu(codes, scales, cols):
    return MxFp4(torch.from_numpy(codes).to(DEV), torch.from_numpy(X.tile_scales(scales)).to(DEV), codes.shape[0], cols)


def _quantized(rows, cols, seed, spread=3.0):
    """A random quantised matrix on the GPU and its values in 64 bits."""
    codes, scales = X.quantize(_matrix(rows, cols, seed, spread).numpy())
    return _to_gpu(codes, scales, cols), X.values(codes, scales, cols)


def _same(q, want_of):
    codes, scales = X.quantize(want_of)
    assert (q.rows, q.cols) == want_of.shape
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    assert np.array_equal(q.scales.cpu().numpy(), X.tile_scales(scales))


def _poisoned(rows, cols):
    q = MxFp4.empty(rows, cols, DEV)
    q.codes.fill_(0x5A)
    q.scales.fill_(0xA5)
    return q


# ---------------------------------------------------------------- quantisation
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,pad,skip", [(1, 1, 0, 0), (1, 4096, 0, 0), (3, 31, 0, 0), (33, 32, 0, 0), (128, 128, 0, 0),
                                                (129, 257, 0, 0), (257, 1000, 8, 0), (100, 333, 13, 0), (64, 96, 16, 8), (40, 72, 5, 3)])
def test_quantize(ctx, kind, rows, cols, pad, skip):
    wide = _matrix(rows, cols + pad + skip, rows + cols).to(TYPES[kind]).to(DEV)
    x = wide[:, skip:skip + cols]
    want = x.double().cpu().numpy()
    r, c = ctx.quantize_mxfp4(x, "both", out=(_poisoned(rows, cols), _poisoned(cols, rows)))
    _same(r, want)
    _same(c, np.ascontiguousarray(want.T))
    _same(ctx.quantize_mxfp4(x, out=_poisoned(rows, cols)), want)
    _same(ctx.quantize_mxfp4(x, "columns", out=_poisoned(cols, rows)), np.ascontiguousarray(want.T))
    assert ctx.sync() == 0


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_quantize_special_values(ctx, kind):
    """Zeros of either sign, infinities and NaN, subnormal and largest numbers, exact powers of two, every tie."""
    t = TYPES[kind]
    info = torch.finfo(t)
    x = torch.randn(70, 80, generator=torch.Generator().manual_seed(1)).to(t)
    x[0] = 0
    x[1] = -0.0
    x[2, 5] = float("inf")
    x[3, 40] = -float("inf")
    x[4, 79] = float("nan")
    x[5] = info.max
    x[6] = -info.max * 0.7
    x[7] = info.tiny
    x[8] = info.smallest_normal * torch.linspace(-1, 1, 80)     # subnormal numbers of the type
    x[9] = info.smallest_normal * info.eps                      # the smallest one
    x[10] = 2.0 ** torch.arange(-10, 6).repeat(5).to(torch.float32)
    x[11] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] * 10)
    x[12] = -x[11]
    x[13] = torch.nextafter(x[11].float(), torch.tensor(9.0)).to(t)
    x[14, 1:] = 0
    x = x.to(DEV)
    want = x.double().cpu().numpy()
    r, c = ctx.quantize_mxfp4(x, "both")
    _same(r, want)
    _same(c, np.ascontiguousarray(want.T))
    v = ctx.dequantize_mxfp4(r, torch.float32).double().cpu().numpy()
    assert np.array_equal(v, X.rounded(want), equal_nan=True)
    assert np.isnan(v[2, :32]).all() and np.isfinite(v[2, 32:]).all() and ctx.sync() == 0


def test_quantize_leaves_the_rest_of_its_buffers(ctx):
    rows, cols = 130, 100
    x = _matrix(rows, cols, 3).float().to(DEV)
    pitch, size = X.blocks(cols) * 16, 2 * 512
    codes = torch.full((rows * pitch + 64,), 0x77, dtype=torch.uint8, device=DEV)
    scales = torch.full((size + 64,), 0x66, dtype=torch.uint8, device=DEV)
    q = MxFp4(codes[:rows * pitch].view(rows, pitch), scales[:size], rows, cols)
    _same(ctx.quantize_mxfp4(x, out=q), x.double().cpu().numpy())
    assert bool((codes[rows * pitch:] == 0x77).all()) and bool((scales[size:] == 0x66).all())


# ---------------------------------------------------------------- values
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 4096, 0), (33, 40, 0), (129, 257, 0), (300, 136, 8), (65, 100, 13)])
def test_dequantize(ctx, kind, rows, cols, pad):
    q, want = _quantized(rows, cols, 5)
    out = torch.full((rows, cols + pad), 3.0, dtype=TYPES[kind], device=DEV)
    got = ctx.dequantize_mxfp4(q, out=out[:, :cols])
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(TYPES[kind]))     # one rounding of the exact value
    assert bool((out[:, cols:] == 3).all()) and ctx.sync() == 0


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_dequantize_every_scale_and_code(ctx, kind):
    codes = np.arange(256, dtype=np.uint8).reshape(1, -1).repeat(256, 0)      # 16 blocks a row hold all pairs of codes
    scales = np.arange(256, dtype=np.uint8).reshape(-1, 1).repeat(16, 1)
    got = ctx.dequantize_mxfp4(_to_gpu(codes, scales, 512), TYPES[kind])
    want = torch.from_numpy(X.values(codes, scales, 512)).float().to(TYPES[kind])   # 6 * 2^127 is infinite in 32 bits too
    assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(got.cpu().isnan(), want.isnan())


# ---------------------------------------------------------------- products
SHAPES = [(1, 1, 1), (1, 16, 32), (2, 33, 31), (16, 128, 64), (17, 100, 33), (32, 130, 256), (33, 257, 500), (64, 96, 1000),
          (65, 129, 300), (100, 1000, 96), (128, 128, 2048), (129, 300, 4103), (256, 256, 512), (257, 513, 1030), (300, 700, 2049),
          (520, 1000, 288), (1, 4096, 4096),
          # more tiles than CTA pairs: both accumulators in turn, a last wave of column halves; long K on few tiles; many
          # narrow tiles, two to an SM
          (2500, 2000, 300), (1300, 4500, 1030), (100, 200, 9000), (20, 30000, 1030)]


def _bound(a, b, K, kind):
    """A 32-bit sum of K exact products, in any order, each addition rounded or cut: at most K * 2^-23 of the sum of their
    magnitudes; then half a step of the result's type."""
    return K * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T) + HALF_STEP[kind] * np.abs(a @ b.T) + 2.0 ** -25


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(ctx, M, N, K, kind):
    (A, a), (B, b) = _quantized(M, K, M + K), _quantized(N, K, N + 7)
    out = torch.full((M, N + 3), 5.0, dtype=TYPES[kind], device=DEV)
    got = ctx.gemm_mxfp4(A, B, TYPES[kind])
    assert ctx.sync() == 0
    c, ref, bound = got.double().cpu().numpy(), a @ b.T, _bound(a, b, K, kind)
    # 16-bit floats end at 65504: rounding to nearest gives an infinity from 65504 + half a step (16) = 65520 on, so one
    # stands, with its sign, for a sum that can be that large, and nothing else is let off its bound
    over = np.isinf(c) & (kind == "f16")
    assert (np.abs(ref) + bound >= 65520)[over].all() and (np.sign(c) == np.sign(ref))[over].all()
    far = np.abs(np.where(over, ref, c) - ref) - bound
    assert far.max() <= 0, (far.max(), np.argwhere(far > 0)[:5])
    ctx.gemm_mxfp4(A, B, out=out[:, :N])                                      # rows further apart, no vector fits
    assert torch.equal(out[:, :N], got) and bool((out[:, N:] == 5).all()) and ctx.sync() == 0


@pytest.mark.parametrize("M,N,K", [(3, 70, 100), (3, 72, 100), (65, 128, 300), (67, 1001, 4103), (300, 520, 1030), (300, 519, 1030),
                                   (2500, 2000, 300)])
def test_product_is_added(ctx, M, N, K):
    (A, a), (B, b) = _quantized(M, K, 1), _quantized(N, K, 2)
    c = torch.randn(M, N + 4, generator=torch.Generator().manual_seed(3)).to(DEV)
    was = c.clone()
    got = ctx.gemm_mxfp4(A, B, out=c[:, :N], accumulate=True)
    ref = was[:, :N].double().cpu().numpy() + a @ b.T
    far = np.abs(got.double().cpu().numpy() - ref) - _bound(a, b, K, "f32") - 2.0 ** -24 * np.abs(ref)
    assert far.max() <= 0 and torch.equal(c[:, N:], was[:, N:]) and ctx.sync() == 0


@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (70, 300, 520), (300, 300, 300)])
def test_a_block_that_is_nan_reaches_its_row_or_column_alone(ctx, M, N, K):
    a, b = _matrix(M, K, 1).numpy(), _matrix(N, K, 2).numpy()
    a[M // 2, K - 1] = np.inf
    b[N - 1, 0] = np.nan
    qa, qb = X.quantize(a), X.quantize(b)
    got = ctx.gemm_mxfp4(_to_gpu(*qa, K), _to_gpu(*qb, K), torch.float32).cpu().numpy()
    want = np.zeros((M, N), dtype=bool)
    want[M // 2] = True
    want[:, N - 1] = True
    assert np.array_equal(np.isnan(got), want) and ctx.sync() == 0


def _whole(rows, cols, seed, exps=(0, 2)):
    """A quantised matrix whose products with another one sum exactly in 32 bits: every value is a multiple of 0.5 and
    at most 6 * 2^1, so a product is a multiple of 0.25 and at most 144; 2^24 of a quarter cover K up to 29127."""
    rng = np.random.default_rng(seed)
    scales = (127 + rng.integers(*exps, (rows, X.blocks(cols)))).astype(np.uint8)
    codes = rng.integers(0, 256, (rows, X.blocks(cols) * 16)).astype(np.uint8)
    if cols % 32:
        full = np.stack([codes & 15, codes >> 4], 2).reshape(rows, -1)
        full[:, cols:] = 0
        codes = full[:, 0::2] | (full[:, 1::2] << 4)
    return _to_gpu(codes, scales, cols), X.values(codes, scales, cols)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_is_exact_where_32_bits_hold_it(ctx, M, N, K):
    (A, a), (B, b) = _whole(M, K, 11), _whole(N, K, 12)
    assert np.array_equal(ctx.gemm_mxfp4(A, B, torch.float32).double().cpu().numpy(), a @ b.T) and ctx.sync() == 0


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_requantised_product(ctx, M, N, K):
    (A, a), (B, b) = _whole(M, K, 21), _whole(N, K, 22)
    _same(ctx.gemm_mxfp4_mxfp4(A, B, out=_poisoned(M, N)), a @ b.T)
    assert ctx.sync() == 0


def test_requantised_product_with_nan_and_zero_rows(ctx):
    a, b = _matrix(70, 96, 4).numpy(), _matrix(200, 96, 5).numpy()
    a[3] = 0
    a[5, 50] = np.nan
    (ca, sa), (cb, sb) = X.quantize(a), X.quantize(b)
    q = ctx.gemm_mxfp4_mxfp4(_to_gpu(ca, sa, 96), _to_gpu(cb, sb, 96))
    s = X.untile_scales(q.scales.cpu().numpy(), 70, 200)
    assert (s[3] == 0).all() and (s[5] == 255).all() and (s[[0, 1, 2, 4, 69]] < 255).all()
    assert (q.codes[[3, 5]].cpu() & 0x77 == 0).all() and ctx.sync() == 0


@pytest.mark.parametrize("M,N", [(0, 8), (8, 0), (0, 0)])
def test_empty_results(ctx, M, N):
    A, B = MxFp4.empty(M, 64, DEV), MxFp4.empty(N, 64, DEV)
    assert ctx.gemm_mxfp4(A, B).shape == (M, N)
    assert ctx.gemm_mxfp4_mxfp4(A, B).rows == M
    assert ctx.quantize_mxfp4(torch.empty(M, N, device=DEV)).rows == M
    assert ctx.dequantize_mxfp4(MxFp4.empty(M, N, DEV)).shape == (M, N) and ctx.sync() == 0


def test_empty_sum(ctx):
    A, B = MxFp4.empty(5, 0, DEV), MxFp4.empty(40, 0, DEV)
    c = torch.full((5, 44), 2.0, device=DEV)
    ctx.gemm_mxfp4(A, B, out=c[:, :40], accumulate=True)
    assert bool((c == 2).all())
    ctx.gemm_mxfp4(A, B, out=c[:, :40])
    assert bool((c[:, :40] == 0).all()) and bool((c[:, 40:] == 2).all())
    q = ctx.gemm_mxfp4_mxfp4(A, B, out=_poisoned(5, 40))
    assert bool((q.codes == 0).all()) and bool((q.scales == 0).all()) and ctx.sync() == 0


# ---------------------------------------------------------------- together, as they are used
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("tokens,n,k", [(1, 64, 32), (130, 200, 328), (300, 520, 600)])
def test_training_step_of_a_layer(ctx, tokens, n, k, kind):
    """y = x w^T and both gradients, all operands quantised along the sums' axes from one reading each, against 64 bits."""
    t = TYPES[kind]
    x, w, dy = (_matrix(*s, 30 + i).to(t).to(DEV) for i, s in enumerate([(tokens, k), (n, k), (tokens, n)]))
    (xq, xt), (wq, wt), (gq, gt) = (ctx.quantize_mxfp4(m, "both") for m in (x, w, dy))
    y = ctx.gemm_mxfp4(xq, wq, t)
    dx = ctx.gemm_mxfp4(gq, wt, t)
    dw = ctx.gemm_mxfp4(gt, xt, torch.float32)
    x, w, dy = (m.double().cpu().numpy() for m in (x, w, dy))
    for got, a, b, kd in ((y, x, w, kind), (dx, dy, w.T, kind), (dw, dy.T, x.T, "f32")):
        a, b = X.rounded(a), X.rounded(b)
        assert (np.abs(got.double().cpu().numpy() - a @ b.T) <= _bound(a, b, a.shape[1], kd)).all()
    assert ctx.sync() == 0


def test_gradients_against_differences(ctx):
    """loss = sum(g * (a b^T)): its differences along single elements of a and b, taken through the product itself, are
    the gradients that the products on column quantisations give.  All values lie on the grid with scale 1 (largest
    magnitude 4 or 6 in every block), so quantisation changes nothing and every sum is exact."""
    rng = np.random.default_rng(8)
    M, N, K = 64, 96, 128

    def grid(r, c):
        v = X.GRID[rng.integers(0, 8, (r, c))] * rng.choice([-1, 1], (r, c))
        v[::32, :] = 6
        v[:, ::32] = 4
        return torch.from_numpy(v).float().to(DEV)
    a, b, g = grid(M, K), grid(N, K), grid(M, N)
    gq, gt = ctx.quantize_mxfp4(g, "both")
    da = ctx.gemm_mxfp4(gq, ctx.quantize_mxfp4(b, "columns"), torch.float32)
    db = ctx.gemm_mxfp4(gt, ctx.quantize_mxfp4(a, "columns"), torch.float32)

    def loss(a, b):
        return float((g.double() * ctx.gemm_mxfp4(ctx.quantize_mxfp4(a), ctx.quantize_mxfp4(b), torch.float32).double()).sum())
    for i, j in ((1, 1), (33, 5), (63, 127)):
        for m, d in ((a, da), (b, db)):
            up, down = m.clone(), m.clone()
            up[i, j], down[i, j] = 3, -2
            ends = [(up, b), (down, b)] if m is a else [(a, up), (a, down)]
            assert (loss(*ends[0]) - loss(*ends[1])) / 5 == float(d[i, j])


def test_chain_of_requantised_products(ctx):
    (A, a), (B, b), (D, d) = _whole(130, 256, 1), _whole(192, 256, 2), _whole(70, 192, 3)
    q = ctx.gemm_mxfp4_mxfp4(A, B)
    got = ctx.gemm_mxfp4(q, D, torch.float32).double().cpu().numpy()
    m = X.rounded(a @ b.T)
    assert (np.abs(got - m @ d.T) <= _bound(m, d, 192, "f32")).all() and ctx.sync() == 0


# ---------------------------------------------------------------- streams, graphs, contexts
def test_another_stream(ctx):
    (A, a), (B, b) = _whole(100, 512, 1), _whole(300, 512, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ctx.gemm_mxfp4(A, B, torch.float32)
        q = ctx.quantize_mxfp4(got)
        v = ctx.dequantize_mxfp4(q, torch.float32)
        assert ctx.sync() == 0
    assert np.array_equal(got.double().cpu().numpy(), a @ b.T)
    assert np.array_equal(v.double().cpu().numpy(), X.rounded(a @ b.T))


def test_two_captured_graphs_replayed_side_by_side(ctx):
    """No workspace is shared: two graphs of one context run at the same time, and again with other inputs."""
    sets = []
    for seed in (1, 2):
        x = _matrix(80, 512, seed).float().to(DEV)
        (W, w) = _whole(600, 512, seed + 10)
        out = torch.empty(80, 600, device=DEV)
        q, r = MxFp4.empty(80, 512, DEV), MxFp4.empty(80, 600, DEV)

        def step(x=x, W=W, out=out, q=q, r=r):
            ctx.quantize_mxfp4(x, out=q)
            ctx.gemm_mxfp4(q, W, out=out)
            ctx.gemm_mxfp4_mxfp4(q, W, out=r)
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        sets.append((x, w, out, q, r, g, torch.cuda.Stream()))
    for turn in range(3):
        for i, (x, *_) in enumerate(sets):
            x.copy_(_matrix(80, 512, 50 + 2 * turn + i).float())
        torch.cuda.synchronize()
        for _ in range(10):
            for *_, g, s in sets:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for x, w, out, q, r, *_ in sets:
            a = X.rounded(x.double().cpu().numpy())
            _same(q, x.double().cpu().numpy())
            assert (np.abs(out.double().cpu().numpy() - a @ w.T) <= _bound(a, w, 512, "f32")).all()
            _same(r, out.double().cpu().numpy())
    assert ctx.sync() == 0


def test_results_do_not_depend_on_the_run(ctx):
    (A, _), (B, _) = _quantized(40, 8192, 1), _quantized(300, 8192, 2)
    first = ctx.gemm_mxfp4(A, B, torch.float32)
    assert all(torch.equal(ctx.gemm_mxfp4(A, B, torch.float32), first) for _ in range(20))


@pytest.mark.parametrize("M,N,K", [(16, 300, 4096), (600, 600, 2048)])
def test_a_wait_that_runs_out_is_reported_and_the_context_survives(M, N, K):
    c = Context(0)
    try:
        (A, a), (B, b) = _whole(M, K, 1), _whole(N, K, 2)
        c.set_debug(3)
        c.gemm_mxfp4(A, B)
        with pytest.raises(Exception, match="status word"):
            c.sync()
        c.set_debug(0)
        assert np.array_equal(c.gemm_mxfp4(A, B, torch.float32).double().cpu().numpy(), a @ b.T) and c.sync() == 0
    finally:
        c.close()


def test_one_matrix_as_both_operands(ctx):
    (A, a) = _whole(300, 500, 1)
    assert np.array_equal(ctx.gemm_mxfp4(A, A, torch.float32).double().cpu().numpy(), a @ a.T) and ctx.sync() == 0


def test_among_other_kernels_without_a_pause(ctx):
    """Launches that start while the one before drains (and hold TMEM then): int8 and 4-bit products of both forms,
    quantisation and values in one stream, each reading what the call before has written."""
    (A, a), (B, b) = _whole(300, 512, 1), _whole(512, 512, 2)
    i8 = torch.randint(-8, 8, (256, 256), dtype=torch.int8, device=DEV)
    want8 = (i8.float() @ i8.float().t()).int()
    outs, ref = [], None
    for _ in range(30):
        c = ctx.gemm_mxfp4(A, B, torch.float32)
        r, t = ctx.quantize_mxfp4(c, "both")
        d = ctx.gemm_mxfp4(r, B, torch.float32)
        e = ctx.gemm_i8_i32(i8, i8)
        q = ctx.gemm_mxfp4_mxfp4(MxFp4(r.codes[:16], r.scales[:2048], 16, 512), B)
        outs.append((c, d, e, ctx.dequantize_mxfp4(q, torch.float32), ctx.dequantize_mxfp4(t, torch.float32)))
    assert ctx.sync() == 0
    m = X.rounded(a @ b.T)
    assert np.array_equal(outs[0][0].double().cpu().numpy(), a @ b.T)
    assert (np.abs(outs[0][1].double().cpu().numpy() - m @ b.T) <= _bound(m, b, 512, "f32")).all()
    assert np.array_equal(outs[0][3].double().cpu().numpy(), X.rounded(outs[0][1][:16].double().cpu().numpy()))
    assert np.array_equal(outs[0][4].double().cpu().numpy(), X.rounded((a @ b.T).T))
    for c, d, e, f, g in outs:
        assert torch.equal(e, want8)
        assert all(torch.equal(x, y) for x, y in zip((c, d, f, g), (outs[0][i] for i in (0, 1, 3, 4))))


def test_bound_calls(ctx):
    """The calls with their arguments converted once, as the other products have them."""
    x = _matrix(70, 300, 1).float().to(DEV)
    (W, w) = _whole(200, 300, 2)
    r, c = _poisoned(70, 300), _poisoned(300, 70)
    out = torch.empty(70, 200, device=DEV)
    both, rows, columns = (ctx.bound_quantize_mxfp4(x, o, way) for o, way in (((r, c), "both"), (r, "rows"), (c, "columns")))
    product, adding = ctx.bound_gemm_mxfp4(r, W, out), ctx.bound_gemm_mxfp4(r, W, out, accumulate=True)
    before = ctx.launch_count
    both()
    _same(r, x.double().cpu().numpy())
    _same(c, np.ascontiguousarray(x.double().cpu().numpy().T))
    x.mul_(-2)
    rows(), columns(), product()
    _same(c, np.ascontiguousarray(x.double().cpu().numpy().T))
    want = ctx.gemm_mxfp4(ctx.quantize_mxfp4(x), W, torch.float32)
    assert torch.equal(out, want)
    adding()
    assert torch.equal(out, 2 * want) and ctx.launch_count == before + 7 and ctx.sync() == 0
    for bind in (lambda: ctx.bound_quantize_mxfp4(x, None), lambda: ctx.bound_gemm_mxfp4(r, W, None)):
        with pytest.raises(ValueError, match="needs an output"):
            bind()
    with pytest.raises(ValueError, match="K differs"):
        ctx.bound_gemm_mxfp4(c, W, out)
    with pytest.raises(ValueError, match="shape or type"):
        ctx.bound_gemm_mxfp4(r, W, out[:69])
    with pytest.raises(ValueError, match="other sizes"):
        ctx.bound_quantize_mxfp4(x, c)


def test_two_streams_at_once(ctx):
    sets = [_whole(m, 1030, m) + _whole(700, 1030, m + 1) for m in (5, 300, 40, 1000)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]
    for _ in range(10):
        for s, (A, _, B, _), g in zip(streams, sets, got):
            with torch.cuda.stream(s):
                g.append(ctx.gemm_mxfp4(A, B, torch.float32))
    torch.cuda.synchronize()
    for (_, a, _, b), g in zip(sets, got):
        assert all(np.array_equal(c.double().cpu().numpy(), a @ b.T) for c in g)
    assert ctx.sync() == 0


@pytest.mark.parametrize("sms", [1, 2, 7, 64])
def test_a_limit_on_the_sms(sms):
    c = Context(0)
    try:
        c.set_cta_limit(sms)
        for M, N, K in ((3, 700, 1030), (100, 300, 2048), (600, 900, 520)):
            (A, a), (B, b) = _whole(M, K, 1), _whole(N, K, 2)
            assert np.array_equal(c.gemm_mxfp4(A, B, torch.float32).double().cpu().numpy(), a @ b.T)
            _same(c.gemm_mxfp4_mxfp4(A, B, out=_poisoned(M, N)), a @ b.T)
        assert c.sync() == 0
    finally:
        c.close()


def test_offsets_past_32_bits(ctx):
    """More than 2^32 elements (2^31 bytes of codes): the last rows are where 32-bit offsets would go wrong."""
    rows, cols = 131100, 33000
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(1))
    r, t = ctx.quantize_mxfp4(x, "both")
    at = torch.tensor([0, 1, 65077, 130175, 131098, 131099], device=DEV)
    want = X.rounded(x[at].double().cpu().numpy())
    v = ctx.dequantize_mxfp4(r)
    assert np.array_equal(v[at].double().cpu().numpy(), want)
    del v
    cols_at = torch.tensor([0, 31, 16001, 32998, 32999], device=DEV)
    want_t = X.rounded(x[:, cols_at].double().cpu().numpy().T)
    del x
    v = ctx.dequantize_mxfp4(t)
    assert np.array_equal(v[cols_at].double().cpu().numpy(), want_t)
    del v, t
    (B, b) = _quantized(8, cols, 3)
    c = ctx.gemm_mxfp4(B, r, torch.float32)                                   # long rows, many of them
    assert (np.abs(c[:, at].double().cpu().numpy() - b @ want.T) <= _bound(b, want, cols, "f32")).all()
    del c, r
    (A, a), (B, b) = _whole(rows, 64, 5), _whole(cols, 64, 6)
    c = ctx.gemm_mxfp4(A, B)                                                  # a result of more than 2^32 elements
    ref = torch.from_numpy(a[at.cpu().numpy()] @ b.T).to(torch.bfloat16)
    assert torch.equal(c[at].cpu(), ref)
    del c
    q = ctx.gemm_mxfp4_mxfp4(A, B)
    v = ctx.dequantize_mxfp4(q)
    assert np.array_equal(v[at].double().cpu().numpy(), X.rounded(a[at.cpu().numpy()] @ b.T)) and ctx.sync() == 0


# ---------------------------------------------------------------- refusals of the Python face
def test_refusals(ctx):
    x = torch.randn(40, 64, device=DEV)
    q, other = ctx.quantize_mxfp4(x), ctx.quantize_mxfp4(torch.randn(8, 32, device=DEV))
    before = ctx.launch_count
    with pytest.raises(ValueError, match="way"):
        ctx.quantize_mxfp4(x, "diagonal")
    with pytest.raises(TypeError, match="float32"):
        ctx.quantize_mxfp4(x.double())
    with pytest.raises(TypeError, match="CUDA tensor"):
        ctx.quantize_mxfp4(x.cpu())
    with pytest.raises(ValueError, match="contiguous"):
        ctx.quantize_mxfp4(x.t())
    with pytest.raises(ValueError, match="overlap"):
        ctx.quantize_mxfp4(x.flatten()[:64].as_strided((4, 32), (8, 1)))
    with pytest.raises(ValueError, match="matrix"):
        ctx.quantize_mxfp4(x[0])
    with pytest.raises(ValueError, match="other sizes"):
        ctx.quantize_mxfp4(x, out=MxFp4.empty(40, 65, DEV))
    with pytest.raises(TypeError, match="MxFp4"):
        ctx.quantize_mxfp4(x, "both", out=(None, MxFp4.empty(64, 40, DEV)))
    with pytest.raises(TypeError, match="MxFp4"):
        ctx.gemm_mxfp4(x, q)
    with pytest.raises(ValueError, match="K differs"):
        ctx.gemm_mxfp4(q, other)
    with pytest.raises(ValueError, match="K differs"):
        ctx.gemm_mxfp4_mxfp4(q, other)
    with pytest.raises(ValueError, match="existing output"):
        ctx.gemm_mxfp4(q, q, accumulate=True)
    with pytest.raises(Exception, match="only f32"):
        ctx.gemm_mxfp4(q, q, out=torch.zeros(40, 40, dtype=torch.bfloat16, device=DEV), accumulate=True)
    with pytest.raises(ValueError, match="shape or type"):
        ctx.gemm_mxfp4(q, q, out=torch.zeros(40, 41, device=DEV))
    with pytest.raises(ValueError, match="shape or type"):
        ctx.gemm_mxfp4(q, q, torch.float32, out=torch.zeros(40, 40, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="bytes for"):
        MxFp4(q.codes, q.scales, 40, 65)
    with pytest.raises(ValueError, match="bytes for"):
        MxFp4(torch.empty(129, 32, dtype=torch.uint8, device=DEV), q.scales, 129, 64)
    with pytest.raises(ValueError, match="negative"):
        MxFp4.empty(-1, 64, DEV)
    with pytest.raises(ValueError, match="contiguous"):
        MxFp4(torch.empty(32, 40, dtype=torch.uint8, device=DEV).t(), q.scales, 40, 64)
    with pytest.raises(TypeError, match="uint8"):
        MxFp4(q.codes, q.scales.float(), 40, 64)
    with pytest.raises(TypeError, match="one device"):
        MxFp4(q.codes, q.scales.cpu(), 40, 64)
    with pytest.raises(TypeError, match="CUDA device"):
        MxFp4.empty(4, 64, "cpu")
    with pytest.raises(Exception, match="16-byte"):
        ctx.dequantize_mxfp4(MxFp4(torch.empty(40 * 32 + 8, dtype=torch.uint8, device=DEV)[8:].view(40, 32), q.scales, 40, 64))
    assert ctx.launch_count == before and ctx.sync() == 0
