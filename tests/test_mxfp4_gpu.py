"""MXFP4 (E2M1 data, one UE8M0 scale per 32 K): the activation quantiser and the block-scaled GEMM against their
definitions in 64 bits.  Data format: op/test/arch_primitives/ptx_mma_fp4.cu:49-53,120-130; scale decoder
op/test/arch_primitives/ptx_mma_fp6.cu:344-351."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def codes_of(y):
    """E2M1 codes of 64-bit values: nearest, of two equally near ones the even code, saturating; sign in bit 3."""
    a = np.abs(y)
    code = np.zeros(y.shape, np.uint8)
    for i in range(1, 8):
        border = (GRID[i - 1] + GRID[i]) / 2
        code[(a >= border) if i % 2 == 0 else (a > border)] = i
    return code | (np.signbit(y).astype(np.uint8) << 3)


def quantise(x):
    """(codes [rows, K], scale bytes [rows, K/32]) of float64 rows."""
    b = x.reshape(x.shape[0], -1, 32)
    a = np.abs(b).max(2)
    bad = ~np.isfinite(a)
    _, e = np.frexp(np.where(bad | (a == 0), 1.0, a))            # a = f * 2^e, f in [0.5, 1)
    s = np.where(bad, 255, np.where(a == 0, 0, np.maximum(e - 3 + 127, 0))).astype(np.uint8)
    y = np.where(bad[:, :, None], 0.0, b) / np.exp2(s.astype(np.float64) - 127)[:, :, None]
    return np.where(bad[:, :, None], 0, codes_of(y)).astype(np.uint8).reshape(x.shape), s


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def blocked(s):
    rows, k32 = s.shape
    out = np.zeros((-(-rows // 128), -(-k32 // 4), 512), np.uint8)
    for r in range(rows):
        for j in range(k32):
            out[r // 128, j // 4, (r % 32) * 16 + (r % 128 // 32) * 4 + j % 4] = s[r, j]
    return out.reshape(-1)


def values(codes, s):
    v = np.concatenate([GRID, -GRID])[codes]
    w = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127))
    return v * w.repeat(32, axis=1)


def case(M, N, K, seed):
    rng = np.random.default_rng(seed)
    a = rng.integers(0, 16, (M, K)).astype(np.uint8)
    b = rng.integers(0, 16, (N, K)).astype(np.uint8)
    sa = rng.integers(121, 134, (M, K // 32)).astype(np.uint8)
    sb = rng.integers(121, 134, (N, K // 32)).astype(np.uint8)
    return a, sa, b, sb


def check_product(out, a, sa, b, sb):
    va, vb = values(a, sa), values(b, sb)
    want = va @ vb.T
    # one rounding to bf16 (2^-8 of the value), and per accumulation step of 64 K an addition whose error is at most 2^-22
    # of the sum of the magnitudes (a truncated 32-bit sum, with the alignment of the step's own products)
    bound = 2.0 ** -8 * np.abs(want) + (a.shape[1] / 64 + 2) * 2.0 ** -22 * (np.abs(va) @ np.abs(vb).T) + 1e-300
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


# few rows (1..128: the streaming kernel, K in one part and split), many rows (the pair kernel, or the streaming one in tiles of
# 128 rows where there are few tiles; three tile widths, one tile a CTA pair and several); K ending inside an instruction's step,
# inside a scale block and inside a slab; rows of the output on every alignment
@pytest.mark.parametrize("shape", [(1, 1, 32), (1, 130, 64), (3, 300, 96), (16, 128, 2048), (17, 257, 2080), (64, 1000, 4096),
                                   (100, 129, 544), (128, 256, 8192), (129, 300, 288), (200, 72, 4128), (333, 513, 1056),
                                   (512, 384, 512), (130, 474, 4128), (600, 129, 8192), (257, 1025, 4096), (400, 262, 96), (290, 131, 64),
                                   (520, 3301, 96), (520, 4704, 64), (1030, 5003, 64), (1030, 10002, 32)])
def test_product_against_64_bits(shape):
    import cudaop_b200 as ops
    M, N, K = shape
    a, sa, b, sb = case(M, N, K, M + N + K)
    out = ops.gemm_mxfp4(dev(pack(a)), dev(sa), dev(pack(b)), dev(sb))
    again = ops.gemm_mxfp4(dev(pack(a)), dev(blocked(sa)), dev(pack(b)), dev(blocked(sb)), blocked=True)
    torch.cuda.synchronize()
    assert ops.status() == 0
    assert out.shape == (M, N) and out.dtype == torch.bfloat16
    assert torch.equal(out, again)
    check_product(out, a, sa, b, sb)


@pytest.mark.parametrize("M", [16, 300])
def test_every_scale_byte_is_used_exactly(M):
    """All codes 1.0, a scale that differs per row and per 32 K: the sums are small integers times powers of two, exact."""
    import cudaop_b200 as ops
    N, K = 160, 512
    one = np.full((1, K), 2, np.uint8)
    sa = (127 + (np.arange(M)[:, None] % 3) + np.arange(K // 32)[None, :] % 4).astype(np.uint8)
    sb = (125 + (np.arange(N)[:, None] % 5) - np.arange(K // 32)[None, :] % 2).astype(np.uint8)
    out = ops.gemm_mxfp4(dev(pack(one.repeat(M, 0))), dev(sa), dev(pack(one.repeat(N, 0))), dev(sb))
    want = 32.0 * (np.exp2(sa.astype(np.float64) - 127) @ np.exp2(sb.astype(np.float64) - 127).T)
    assert torch.equal(out, torch.from_numpy(want).cuda().bfloat16())


@pytest.mark.parametrize("M", [5, 200])
def test_a_nan_scale_reaches_its_row_alone(M):
    import cudaop_b200 as ops
    N, K = 140, 320
    a, sa, b, sb = case(M, N, K, 9)
    a[3, 64:96] = 2
    sa[3, 2] = 255
    out = ops.gemm_mxfp4(dev(pack(a)), dev(sa), dev(pack(b)), dev(sb))
    keep = np.arange(M) != 3
    assert out[3].isnan().all() and not out[torch.from_numpy(keep).cuda()].isnan().any()
    check_product(out[torch.from_numpy(keep).cuda()], a[keep], sa[keep], b, sb)


@pytest.mark.parametrize("shape", [(1, 32), (1, 8192), (3, 96), (33, 160), (127, 128), (128, 2080), (130, 4096), (1000, 1056), (2049, 2048)])
def test_quantiser_is_exact(shape):
    import cudaop_b200 as ops
    rows, cols = shape
    g = torch.Generator().manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g).float())).bfloat16()
    x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.0]).bfloat16()      # every tie of the format
    if rows > 1:
        x[1, :32] = 0
        x[-1, -32:] = 0
        x[-1, -1] = 2.0 ** -133                                                            # the smallest bf16
    q, sf = ops.quant_rows_mxfp4(x.cuda())
    torch.cuda.synchronize()
    codes, s = quantise(x.double().numpy())
    assert np.array_equal(q.cpu().numpy(), pack(codes))
    assert np.array_equal(sf.cpu().numpy(), blocked(s))


def test_quantiser_on_values_that_are_not_finite_and_on_extremes():
    import cudaop_b200 as ops
    x = torch.ones(6, 96, dtype=torch.bfloat16)
    x[0, 5] = float("nan")
    x[1, 40] = float("inf")
    x[2, 95] = -float("inf")
    x[3, :] = torch.finfo(torch.bfloat16).max
    x[4, :] = torch.finfo(torch.bfloat16).tiny
    x[5, 33] = -float("nan")
    q, sf = ops.quant_rows_mxfp4(x.cuda())
    codes, s = quantise(x.double().numpy())
    assert s[0, 0] == 255 and s[1, 1] == 255 and s[2, 2] == 255 and (s == 255).sum() == 4
    assert np.array_equal(q.cpu().numpy(), pack(codes)) and np.array_equal(sf.cpu().numpy(), blocked(s))
    # the NaN scale carries on into the product of its row
    wq, wsf = ops.quant_rows_mxfp4(torch.ones(40, 96, dtype=torch.bfloat16, device="cuda"))
    out = ops.gemm_mxfp4(q, sf, wq, wsf, blocked=True)
    assert out[[0, 1, 2, 5]].isnan().all() and not out[4].isnan().any()


@pytest.mark.parametrize("M", [2, 260])
def test_quantised_layer_on_a_side_stream_and_in_a_graph(M):
    """Quantise and multiply as they are used together: on another stream, and captured and replayed on new inputs."""
    import cudaop_b200 as ops
    g = torch.Generator().manual_seed(M)
    K, N = 1088, 333
    w = torch.randn(N, K, generator=g).bfloat16()
    xs = [torch.randn(M, K, generator=g).bfloat16() for _ in range(3)]
    wq, wsf = ops.quant_rows_mxfp4(w.cuda())

    def layer(x):
        q, sf = ops.quant_rows_mxfp4(x)
        return ops.gemm_mxfp4(q, sf, wq, wsf, blocked=True)
    cb, sb = quantise(w.double().numpy())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = layer(xs[0].cuda())
    side.synchronize()
    ca, sa = quantise(xs[0].double().numpy())
    check_product(out, ca, sa, cb, sb)
    static = xs[0].cuda()
    graph = torch.cuda.CUDAGraph()
    layer(static)
    with torch.cuda.graph(graph):
        held = layer(static)
    for x in xs[1:]:
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        ca, sa = quantise(x.double().numpy())
        check_product(held, ca, sa, cb, sb)
    assert ops.status() == 0


def test_weights_quantised_right_before_their_product():
    """The product must see operands that the kernel just in front of it wrote, weights included."""
    import cudaop_b200 as ops
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, 4096, generator=g).bfloat16()
    for i in range(3):
        w = torch.randn(2048, 4096, generator=g).bfloat16()
        q, sf = ops.quant_rows_mxfp4(x.cuda())
        wq, wsf = ops.quant_rows_mxfp4(w.cuda())
        out = ops.gemm_mxfp4(q, sf, wq, wsf, blocked=True)
        ca, sa = quantise(x.double().numpy())
        cb, sb = quantise(w.double().numpy())
        check_product(out, ca, sa, cb, sb)


@pytest.mark.parametrize("M", [3, 128])
def test_more_columns_than_a_grid_has_rows_of_clusters(M):
    """N beyond 65535 tiles of 128 columns, with few rows of A."""
    import cudaop_b200 as ops
    N, K = 65535 * 128 + 200, 32
    g = torch.Generator(device="cuda").manual_seed(M)
    a, sa, _, _ = case(M, 1, K, M)
    bq = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device="cuda")
    sb = torch.randint(121, 134, (N, 1), generator=g, dtype=torch.uint8, device="cuda")
    out = ops.gemm_mxfp4(dev(pack(a)), dev(sa), bq, sb)
    va = torch.from_numpy(values(a, sa)).cuda()
    grid = torch.from_numpy(np.concatenate([GRID, -GRID])).cuda()
    worst = 0.0
    for n0 in range(0, N, 1 << 20):
        codes = torch.stack((bq[n0:n0 + (1 << 20)] & 15, bq[n0:n0 + (1 << 20)] >> 4), 2).flatten(1).int()
        vb = grid[codes] * torch.exp2(sb[n0:n0 + (1 << 20)].double() - 127)
        want = va @ vb.T
        bound = 2.0 ** -8 * want.abs() + 3 * 2.0 ** -22 * (va.abs() @ vb.abs().T) + 1e-300
        worst = max(worst, float(((out[:, n0:n0 + (1 << 20)].double() - want).abs() / bound).max()))
    assert ops.status() == 0 and worst <= 1.0, worst


def test_refusals():
    import cudaop_b200 as ops
    a = torch.zeros((128, 48), dtype=torch.uint8, device="cuda")
    s = torch.zeros((128, 3), dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError):
        ops.gemm_mxfp4(a[:, :40].contiguous(), s, a[:, :40].contiguous(), s)         # K % 32
    with pytest.raises(ValueError):
        ops.gemm_mxfp4(a, s[:, :2].contiguous(), a, s)                                 # scale shape
    with pytest.raises(ValueError):
        ops.gemm_mxfp4(a, s.view(-1), a, s.view(-1), blocked=True)                     # blocked scales pad to 128 K
    with pytest.raises(ValueError):
        ops.gemm_mxfp4(a, s, a.cpu(), s)                                               # device
    with pytest.raises(ValueError):
        ops.gemm_mxfp4(a[:, ::2], s, a[:, ::2], s)                                     # not contiguous
    with pytest.raises(ValueError):
        ops.quant_rows_mxfp4(torch.zeros((4, 48), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        ops.quant_rows_mxfp4(torch.zeros((4, 64), dtype=torch.float16, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.quant_rows_mxfp4(torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()


def test_the_kernel_before_does_not_count_against_the_wait_limit():
    """A product launched beside a quantiser that runs longer than the limit of the device's waits."""
    import cudaop_b200 as ops
    L = ops.lib()
    a, sa, b, sb = case(5, 300, 2080, 9)
    args = [dev(pack(a)), dev(sa), dev(pack(b)), dev(sb)]
    blocks = [args[0], ops.mxfp8_swizzle_sf(args[1], 2080), args[2], ops.mxfp8_swizzle_sf(args[3], 2080)]
    want = ops.gemm_mxfp4(*blocks, blocked=True)
    big = torch.zeros((1 << 17, 1 << 14), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    assert L.b200q_set_wait_limit_ms(0, 1) == 0
    try:
        for _ in range(3):
            ops.quant_rows_mxfp4(big)
            got = ops.gemm_mxfp4(*blocks, blocked=True)
            torch.cuda.synchronize()
            assert ops.status() == 0 and torch.equal(got, want)
    finally:
        L.b200q_set_wait_limit_ms(0, 2000)


def test_sizes_that_pass_32_bits_are_refused():
    """Cut to 32 bits, 2^32 + 64 columns would be 64, and all behind them stay unwritten."""
    import cudaop_b200 as ops
    x = torch.empty((1, 2 ** 32 + 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ops.quant_rows_mxfp4(x)
    with pytest.raises(ValueError):
        ops.quant_rows_e4m3(x)
    del x
    for half in (2 ** 30 + 16, 2 ** 31 + 16):                        # K = 2^31 + 32 and 2^32 + 32
        a = torch.empty((1, half), dtype=torch.uint8, device="cuda")
        s = torch.empty((1, 2 * half // 32), dtype=torch.uint8, device="cuda")
        with pytest.raises(ValueError):
            ops.gemm_mxfp4(a, s, a, s)
        del a, s
    torch.cuda.synchronize()
    assert ops.status() == 0
