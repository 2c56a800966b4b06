"""Matrices in four bits against a plain 64-bit implementation: the codes and scales exactly, products within what 32-bit sums allow."""
import pytest
import torch

import plain_four_bits as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMATS = ["nvfp4", "mxfp4"]


def ops():
    from libllm_b200.csrc import ops as o
    return o


def rows_like(rows, cols, seed, dtype=torch.bfloat16, spread=6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-spread, spread, (rows, 1), generator=g).float())
    x[:, torch.rand(cols, generator=g) < 0.02] *= 30
    return x.to(dtype)


def same_values(x, format, got):
    # An nvfp4 scale may be rounded up, so that a value within 3 % of the type's largest stands for more than the type holds: 255/256 2^128 has the
    # row scale 2^117 and the block scale 340 -> 352, and 6 * 352 * 2^117 = 1.03 * 2^128 is infinite in 32 bits.  All else is exact.
    ref = P.values(x, format).to(got.dtype).double()
    assert torch.equal(got.double().cpu(), ref), f"{(got.double().cpu() != ref).sum()} of {ref.numel()} values differ"


# ---------------------------------------------------------------- into four bits and back
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 17), (5, 31), (2, 33), (129, 255), (7, 256), (4, 257), (131, 500), (33, 1000), (2, 2048),
                                       (3, 2049), (5, 4097), (2, 8200), (3, 16384), (2, 16400), (1, 40001)])
def test_values_are_the_nearest(format, dtype, rows, cols):
    x = rows_like(rows, cols, rows * 1000 + cols, dtype)
    q = ops().fp4_quantize(x.to(DEV), format)
    same_values(x, format, ops().fp4_dequantize(q))
    same_values(x, format, ops().fp4_dequantize(q, torch.bfloat16))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(40, 130), (40, 300), (40, 777), (7, 1501), (2500, 1501), (3, 2600), (3, 5001), (3, 9001), (3, 20001), (2, 33000)])
def test_rows_that_start_between_16_bytes(format, dtype, rows, cols):
    """Read from, and brought back to, columns 1 and on of a wider tensor, whose border keeps what it had."""
    wide = rows_like(rows, cols + 2, rows + cols, dtype).to(DEV)
    x = wide[:, 1:cols + 1]
    q = ops().fp4_quantize(x, format)
    ref = ops().fp4_quantize(x.contiguous(), format)                    # (scales behind the last row are nobody's)
    assert torch.equal(q.codes, ref.codes) and torch.equal(q.row_scale, ref.row_scale)
    for to in (torch.float32, torch.bfloat16):
        back = torch.full((rows, cols + 2), 7.0, dtype=to, device=DEV)
        ops().fp4_dequantize(q, out=back[:, 1:cols + 1])
        same_values(x.cpu(), format, back[:, 1:cols + 1])
        assert (back[:, 0] == 7).all() and (back[:, -1] == 7).all()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_halves_go_to_the_even_code_under_every_scale(format, dtype):
    """Values at, just below and just above every border, under all the scales that the format's blocks can have."""
    borders = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5], dtype=torch.float64)
    b, blocks = P.BLOCK[format], []
    step = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -22
    for e in range(-4, 5):
        for m in range(8, 16):
            s = m / 8 * 2.0 ** e if format == "nvfp4" else 2.0 ** e
            near = torch.cat([borders * s * f for f in (1, 1 - step, 1 + step, 1 - 2 * step, 1 + 2 * step)])
            block = torch.zeros(2 * b, dtype=torch.float64)
            block[1:b] = near[:b - 1]
            block[b + 1:2 * b] = near.flip(0)[:b - 1]
            block[0] = block[b] = 6 * s
            blocks.append(block * (-1 if m % 2 else 1))
    x = torch.cat(blocks)[None].to(dtype)
    x = torch.cat([x, -x, x * 2.0 ** -40, x * 2.0 ** 60])
    same_values(x, format, ops().fp4_dequantize(ops().fp4_quantize(x.to(DEV), format)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_numbers_next_to_every_border_under_every_e4m3_scale(dtype):
    """A row of 1,536 at most has the scale 1, so that a block of 6 s at most has the scale s: every e4m3 number up to 256."""
    borders = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5], dtype=torch.float64)
    scales = [m * 2.0 ** -9 for m in range(1, 8)] + [(8 + m) / 8 * 2.0 ** e for e in range(-6, 8) for m in range(8)] + [256.0]
    blocks = [torch.zeros(16)]
    blocks[0][3] = 1536
    for s in scales:
        t = (borders * s).to(dtype)                        # exact: seven bits at most
        assert torch.equal(t.double(), borders * s)
        bits = t.view(torch.int16 if dtype == torch.bfloat16 else torch.int32)
        below, above = (bits - 1).view(dtype).float(), (bits + 1).view(dtype).float()
        for near in (torch.cat([below, t.float()]), torch.cat([above, -t.float()]), torch.cat([-below, -above])):
            block = torch.zeros(16)
            block[0] = 6 * s
            block[1:15] = near
            blocks.append(block)
    x = torch.cat(blocks)[None]
    x = torch.cat([x, -x, x * 2.0 ** -60, x * 2.0 ** 90]).to(dtype)
    code, scale, row = P.quantize(x, "nvfp4")
    assert set(scale[0, 1:].flatten().tolist()) == set(scales) and row[0, 0] == 1
    same_values(x, "nvfp4", ops().fp4_dequantize(ops().fp4_quantize(x.to(DEV), "nvfp4")))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zeros_and_the_ends_of_the_range(format, dtype):
    top = torch.finfo(dtype).max
    x = torch.zeros(8, 96, dtype=dtype)
    x[1, 5] = top
    x[2, :48] = torch.finfo(dtype).tiny
    x[3, 7], x[3, 40] = 2.0 ** -133, -2.0 ** -130          # below the normal numbers
    x[4, 0], x[4, 50], x[4, 51], x[4, 90] = 1.0, 2.0 ** -14, 2.0 ** -18, 2.0 ** -30   # blocks far below the row's largest
    x[5] = -0.0
    x[6, 0], x[6, 20], x[6, 95] = -top, 1.0, 2.0 ** 100
    x[7] = torch.linspace(-3, 3, 96)
    same_values(x, format, ops().fp4_dequantize(ops().fp4_quantize(x.to(DEV), format)))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_row_that_is_not_finite_is_nan_and_the_others_are_as_ever(format, bad):
    o, x, w = ops(), rows_like(5, 300, 1), rows_like(140, 300, 2)
    x[2, 299] = bad
    w[130, 0] = bad
    qx, qw = o.fp4_quantize(x.to(DEV), format), o.fp4_quantize(w.to(DEV), format)
    got = o.fp4_dequantize(qx).cpu()
    assert got[2].isnan().all()
    keep = [0, 1, 3, 4]
    same_values(x[keep], format, got[keep])
    y = o.fp4_gemm(qx, qw).cpu()
    o.check_tc_status()
    assert y[2].isnan().all() and y[:, 130].isnan().all()
    others = [i for i in range(140) if i != 130]
    assert y[keep][:, others].isfinite().all()


@pytest.mark.parametrize("format", FORMATS)
def test_rows_cut_out_of_wider_ones_and_a_matrix_filled_again(format):
    o = ops()
    wide = rows_like(20, 400, 3).to(DEV)
    for at, cols in ((0, 200), (8, 200), (3, 129), (1, 320)):
        x = wide[::2, at:at + cols]
        same_values(x.cpu(), format, o.fp4_dequantize(o.fp4_quantize(x, format)))
    q = o.fp4_quantize(wide, format)
    again = rows_like(20, 400, 4).to(DEV)
    assert o.fp4_quantize(again, format, out=q) is q
    out = torch.full((40, 500), 7.0, device=DEV)
    o.fp4_dequantize(q, out=out[::2, 10:410])
    same_values(again.cpu(), format, out[::2, 10:410])
    assert (out[1::2] == 7).all() and (out[:, :10] == 7).all() and (out[:, 410:] == 7).all()
    one = wide[:1].expand(5, 400)                              # a row stride of 0
    same_values(one.cpu(), format, o.fp4_dequantize(o.fp4_quantize(one, format)))


@pytest.mark.parametrize("format", FORMATS)
def test_codes_and_scales_lie_where_they_are_said_to(format):
    x = rows_like(300, 700, 5)
    q = ops().fp4_quantize(x.to(DEV), format)
    code, scale, row = P.quantize(x, format)
    got = q.codes.cpu()
    assert got.shape == (300, 352)
    low, high = (got & 15).long(), (got >> 4).long()
    nibbles = torch.stack([low, high], 2).reshape(300, -1)
    kinds = torch.cat([P.KINDS, -P.KINDS])
    assert torch.equal(kinds[nibbles][:, :700], code.reshape(300, -1)[:, :700]) and (nibbles[:, 700:] & 7 == 0).all()
    tiles = q.scales.cpu().view(3, -1, 32, 4, 4)                # row tile, four blocks, row % 32, row / 32, block
    by_row = tiles.permute(0, 3, 2, 1, 4).reshape(384, -1)[:300].long()
    e = (by_row - 127).double()
    decoded = torch.pow(2.0, e) if format == "mxfp4" else by_row.to(torch.uint8).view(torch.float8_e4m3fn).double()
    n = scale.shape[1]
    assert torch.equal(decoded[:, :n], scale[:, :, 0]) and (by_row[:, n:] == 0).all()
    assert torch.equal(q.row_scale.cpu().double(), row[:, 0])


# ---------------------------------------------------------------- the product
def check_product(M, N, K, format, out_dtype, seed, x=None, w=None):
    """A term is exact in 32 bits; a sum of K terms in 32 bits is off by at most K 2^-23 of the sum of magnitudes, one truncation a term, whatever
    its order, and a result in bfloat16 by half a step of its own, 2^-9 2 = 2^-8."""
    o = ops()
    x = rows_like(M, K, seed) if x is None else x
    w = (rows_like(N, K, seed + 1, spread=2) * 0.02).to(torch.bfloat16) if w is None else w
    got = o.fp4_gemm(o.fp4_quantize(x.to(DEV), format), o.fp4_quantize(w.to(DEV), format), out_dtype=out_dtype).double().cpu()
    o.check_tc_status()
    a, b = P.values(x, format), P.values(w, format)
    ref, size = a @ b.T, a.abs() @ b.abs().T
    tol = size * K * 2.0 ** -23 + (ref.abs() * 2.0 ** -8 if out_dtype == torch.bfloat16 else 0)
    assert got.shape == (M, N)
    far = (got - ref).abs() - tol
    assert (far <= 0).all(), f"{int((far > 0).sum())} of {far.numel()} off, worst {float(far.max()):.3e} of {float(ref.abs().max()):.3e}"
    return float((got - ref).norm() / ref.norm())


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 64), (1, 130, 256), (3, 7, 100), (8, 300, 512), (16, 128, 257), (17, 129, 300), (32, 500, 1024),
                                   (33, 64, 96), (64, 256, 2048), (65, 127, 1500), (128, 384, 511), (129, 200, 768), (192, 128, 256), (193, 300, 400),
                                   (320, 129, 1280), (385, 1000, 640), (700, 513, 300), (256, 192, 256), (257, 193, 511), (1000, 1, 64), (511, 576, 2048), (1030, 2000, 500)])
def test_product(format, M, N, K):
    check_product(M, N, K, format, torch.float32, M + N + K)
    check_product(M, N, K, format, torch.bfloat16, M + N + K)


@pytest.mark.parametrize("format", FORMATS)
def test_product_of_whole_numbers_is_exact(format):
    """Codes and scales chosen so that every sum is a whole number below 2^24: any misplaced code, block scale or row scale shows."""
    g = torch.Generator().manual_seed(9)
    M, N, K = 200, 260, 640
    b = P.BLOCK[format]

    def matrix(rows):
        code = torch.tensor([0., 1, 2, 3, 4, 6])[torch.randint(0, 6, (rows, K // b, b), generator=g)]
        code[:, :, 0] = 6                                    # the block's scale is then the power of two beside it
        sign = torch.where(torch.rand(rows, K // b, b, generator=g) < 0.5, -1.0, 1.0)
        return (code * sign * torch.exp2(torch.randint(0, 3, (rows, K // b, 1), generator=g).float())).reshape(rows, K)
    x, w = matrix(M), matrix(N)
    o = ops()
    qx, qw = o.fp4_quantize(x.to(DEV), format), o.fp4_quantize(w.to(DEV), format)
    assert torch.equal(o.fp4_dequantize(qx).cpu(), x) and torch.equal(o.fp4_dequantize(qw).cpu(), w)
    assert torch.equal(o.fp4_gemm(qx, qw).cpu().double(), x.double() @ w.double().T)
    o.check_tc_status()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M", [37, 300, 1100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_into_rows_of_a_wider_result(format, M, dtype):
    o = ops()
    N = 250
    x, w = rows_like(M, 300, 1), rows_like(N, 300, 2)
    qx, qw = o.fp4_quantize(x.to(DEV), format), o.fp4_quantize(w.to(DEV), format)
    want = o.fp4_gemm(qx, qw, out_dtype=dtype)
    for at, wide in ((7, 400), (8, 400), (8, 401), (0, 250)):             # rows on 16 bytes and not
        out = torch.full((2 * M, wide), 3.0, device=DEV, dtype=dtype)
        o.fp4_gemm(qx, qw, out=out[::2, at:at + N])
        assert torch.equal(out[::2, at:at + N], want)
        assert (out[1::2] == 3).all() and (out[:, :at] == 3).all() and (out[:, at + N:] == 3).all()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("M,N", [(300, 4099), (1301, 1000), (513, 2560)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_into_rows_of_a_wider_result(format, M, N, dtype):
    """Tiles of two SMs, whose result leaves by TMA where rows start on 16 bytes: whatever hangs over the last token or feature stays as it was."""
    o = ops()
    x, w = rows_like(M, 300, 1), rows_like(N, 300, 2)
    qx, qw = o.fp4_quantize(x.to(DEV), format), o.fp4_quantize(w.to(DEV), format)
    a, b = P.values(x, format), P.values(w, format)
    ref = a @ b.T
    tol = a.abs() @ b.abs().T * 300 * 2.0 ** -23 + (ref.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else 0)     # as check_product
    for at, wide in ((7, N + 21), (8, (N + 39) // 8 * 8), (8, N + 14), (0, N)):
        out = torch.full((2 * M, wide), 3.0, device=DEV, dtype=dtype)
        o.fp4_gemm(qx, qw, out=out[::2, at:at + N])
        assert ((out[::2, at:at + N].double().cpu() - ref).abs() <= tol).all()
        assert (out[1::2] == 3).all() and (out[:, :at] == 3).all() and (out[:, at + N:] == 3).all()


@pytest.mark.parametrize("format", FORMATS)
def test_a_tokens_result_does_not_hang_on_the_others(format):
    o = ops()
    x, w = rows_like(250, 700, 1).to(DEV), rows_like(300, 700, 2).to(DEV)
    qw = o.fp4_quantize(w, format)
    whole = o.fp4_gemm(o.fp4_quantize(x, format), qw)
    for n in (1, 5, 16, 20, 40, 100, 128, 129, 200):
        assert torch.equal(o.fp4_gemm(o.fp4_quantize(x[:n], format), qw), whole[:n])


@pytest.mark.parametrize("M", [5, 100, 400])
@pytest.mark.parametrize("up,down", [(120, -120), (-120, 120), (126, -126), (55, 55), (-60, -60), (-70, -50), (100, -30), (-124, 0)])
def test_rows_at_the_ends_of_the_range(M, up, down):
    """Scales at opposite ends of the range cancel; at the same end what can be held is held (terms of 2^-20 and more, 2^40 at most)."""
    o = ops()
    K, N = 300, 150
    x, w = rows_like(M, K, 1, spread=1).double() * 2.0 ** up, rows_like(N, K, 2, spread=1).double() * 2.0 ** down
    x, w = (x.clamp(-3e38, 3e38).to(torch.bfloat16), w.clamp(-3e38, 3e38).to(torch.bfloat16))
    got = o.fp4_gemm(o.fp4_quantize(x.to(DEV)), o.fp4_quantize(w.to(DEV))).double().cpu()
    o.check_tc_status()
    a, b = P.values(x, "nvfp4"), P.values(w, "nvfp4")
    ref, size = a @ b.T, a.abs() @ b.abs().T
    tol = size * (K + 2) * 2.0 ** -23 + 2.0 ** -149
    assert ((got - ref).abs() <= tol).all(), f"worst {float(((got - ref).abs() / tol).max()):.2f} of what is allowed"


def test_nothing_to_do():
    o = ops()
    none = o.fp4_quantize(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV))
    some = o.fp4_quantize(rows_like(4, 64, 1).to(DEV))
    assert o.fp4_dequantize(none).shape == (0, 64) and none.codes.shape == (0, 32)
    assert o.fp4_gemm(none, some).shape == (0, 4) and o.fp4_gemm(some, none).shape == (4, 0)


def test_on_another_stream_and_captured():
    """The whole chain in a graph, replayed with other rows, on a stream of its own."""
    o = ops()
    x, w = rows_like(6, 512, 1).to(DEV), rows_like(400, 512, 2).to(DEV)
    other = rows_like(6, 512, 3).to(DEV)
    qw = o.fp4_quantize(w)
    want, want2 = o.fp4_gemm(o.fp4_quantize(x), qw), o.fp4_gemm(o.fp4_quantize(other), qw)
    q, out, held = o.Fp4Matrix(6, 512, "nvfp4", DEV), torch.empty(6, 400, device=DEV), x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o.fp4_gemm(o.fp4_quantize(held, out=q), qw, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            o.fp4_gemm(o.fp4_quantize(held, out=q), qw, out=out)
        s.synchronize()
        out.zero_()
        graph.replay()
        s.synchronize()
        assert torch.equal(out, want)
        held.copy_(other)
        graph.replay()
        s.synchronize()
        assert torch.equal(out, want2)


def test_products_behind_products_read_what_the_last_one_left():
    """Quantisation, product, quantisation of the result, product: every kernel starts while the one before it drains."""
    o = ops()
    x, w = rows_like(20, 256, 1).to(DEV), (rows_like(256, 256, 2, spread=1) * 0.1).to(DEV)
    for format in FORMATS:
        y = x
        for _ in range(4):
            qw = o.fp4_quantize(w, format)
            z = o.fp4_gemm(o.fp4_quantize(y, format), qw, out_dtype=torch.bfloat16)
            torch.cuda.synchronize()
            again = o.fp4_gemm(o.fp4_quantize(y, format), qw, out_dtype=torch.bfloat16)
            torch.cuda.synchronize()
            assert torch.equal(z, again)
            y = z
        fast = x
        for _ in range(4):
            fast = o.fp4_gemm(o.fp4_quantize(fast, format), o.fp4_quantize(w, format), out_dtype=torch.bfloat16)
        assert torch.equal(fast, y)


def test_two_streams_at_once():
    """Products, parts of K among them, and their rows on two streams: nothing is shared between calls."""
    o = ops()
    sizes = [(5, 2048, 4096), (300, 700, 512), (20, 1000, 8192), (100, 600, 1024)]
    xs = [rows_like(M, K, i).to(DEV) for i, (M, _, K) in enumerate(sizes)]
    ws = [o.fp4_quantize(rows_like(N, K, 10 + i, spread=2).to(DEV)) for i, (_, N, K) in enumerate(sizes)]
    want = [o.fp4_gemm(o.fp4_quantize(x), w) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                for x, w in zip(xs[k::2], ws[k::2]):
                    got[k].append(o.fp4_gemm(o.fp4_quantize(x), w))
    torch.cuda.synchronize()
    for k in range(2):
        for i, y in enumerate(got[k]):
            assert torch.equal(y, want[k + 2 * (i % 2)])
    o.check_tc_status()


def test_offsets_beyond_32_bits():
    """Rows that lie 2^31 elements and more apart, in and out."""
    o = ops()
    far = 2 ** 31 + 2 ** 27
    x, w = rows_like(2, 500, 1), rows_like(300, 500, 2)
    room = torch.zeros(far + 1024, dtype=torch.bfloat16, device=DEV)
    rows = room.as_strided((2, 500), (far, 1))
    rows.copy_(x)
    q, qw = o.fp4_quantize(rows), o.fp4_quantize(w.to(DEV))
    same_values(x, "nvfp4", o.fp4_dequantize(q))
    rows.zero_()
    o.fp4_dequantize(q, out=rows)
    same_values(x, "nvfp4", rows)
    want = o.fp4_gemm(q, qw, out_dtype=torch.bfloat16)
    out = room.as_strided((2, 300), (far, 1))
    o.fp4_gemm(q, qw, out=out)
    assert torch.equal(out, want)
    # a prompt's rows: the last of 300 lies more than 2^31 elements from the first
    step = far // 299 // 8 * 8
    x = rows_like(300, 500, 3).to(DEV)
    q = o.fp4_quantize(x)
    want = o.fp4_gemm(q, qw, out_dtype=torch.bfloat16)
    for at in (0, 3):
        room.zero_()
        out = room[at:].as_strided((300, 300), (step - 4, 1)) if at else room.as_strided((300, 300), (step, 1))
        o.fp4_gemm(q, qw, out=out)
        assert torch.equal(out, want) and int((room != 0).sum()) == int((want != 0).sum())


# ---------------------------------------------------------------- several tiles to a CTA
def whole(rows, K, format, seed, scale=None):
    """Bfloat16 rows that four bits hold as they are, made on the device: whole numbers up to 6 x 2^2 times the row's power of two (2^scale, or one of eight).
    The sum over K of the products of two such rows is a whole number below (6 x 4)^2 K times the two powers: exact in 32 bits for K below 29,000, in any
    order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    b = P.BLOCK[format]
    n = -(-K // b)
    kinds = torch.tensor([0., 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], device=DEV, dtype=torch.bfloat16)
    code = kinds[torch.randint(0, 11, (rows, n, b), generator=g, device=DEV, dtype=torch.int32)]
    code[:, :, 0] = 6                                        # the block's scale is then the power of two beside it
    code *= torch.exp2(torch.randint(0, 3, (rows, n, 1), generator=g, device=DEV).float()).bfloat16()
    e = torch.randint(-4, 4, (rows, 1, 1), generator=g, device=DEV).float() if scale is None else torch.full((rows, 1, 1), float(scale), device=DEV)
    return (code * torch.exp2(e).bfloat16()).reshape(rows, -1)[:, :K].contiguous()


def same_product(M, N, K, format, dtype, seed, x_scale=None, w_scale=None, times=1):
    """Every element equals the 64-bit product's, narrowed to the result's type."""
    o = ops()
    x, w = whole(M, K, format, seed, x_scale), whole(N, K, format, seed + 1, w_scale)
    qx, qw = o.fp4_quantize(x, format), o.fp4_quantize(w, format)
    want = (x.double() @ w.double().T).to(dtype)
    for _ in range(times):
        out = torch.full((M, N), 7.0, dtype=dtype, device=DEV)
        o.fp4_gemm(qx, qw, out=out)
        o.check_tc_status()
        wrong = out != want
        assert not wrong.any(), f"{int(wrong.sum())} of {M * N} elements differ, the first at {wrong.nonzero()[0].tolist()}"


@pytest.mark.parametrize("M,N,K", [(1030, 16384, 256), (2100, 4099, 256), (600, 16384, 700), (20000, 256, 256), (19200, 1030, 100), (2049, 6000, 2304),
                                   (600, 128256, 256)])
@pytest.mark.parametrize("format", FORMATS)
def test_prompts_into_32_bits_with_several_tiles_to_two_sms(format, M, N, K):
    """Boxes on their way out lie in two buffers that the next tile writes again: last token tiles that leave warps without tokens, features of which a
    warp's last box is not there (N % 96 in 64 .. 95) or hangs over."""
    same_product(M, N, K, format, torch.float32, M + N + K, times=3)


@pytest.mark.parametrize("M,N,K", [(1030, 16384, 256), (1030, 16384, 1280), (2100, 4099, 256), (2100, 4099, 1280), (2049, 6000, 2304), (300, 40000, 700),
                                   (20000, 256, 500), (2048, 16384, 2048)])
@pytest.mark.parametrize("format", FORMATS)
def test_prompts_with_several_tiles_to_two_sms(format, M, N, K):
    """Both accumulators, the ring and the places of scales used again from tile to tile: one, two, three, five, eight and nine stages to a tile."""
    same_product(M, N, K, format, torch.bfloat16, M + N + K)
    same_product(M, N, K, format, torch.float32, M + N + K + 7)


@pytest.mark.parametrize("M,N,K", [(1, 40000, 256), (8, 40000, 2048), (16, 50257, 1111), (17, 40000, 1280), (33, 44444, 700), (64, 40000, 2304),
                                   (100, 40000, 256), (128, 60000, 1500)])
@pytest.mark.parametrize("format", FORMATS)
def test_few_tokens_with_several_tiles_to_an_sm(format, M, N, K):
    same_product(M, N, K, format, torch.float32, M + N + K)
    same_product(M, N, K, format, torch.bfloat16, M + N + K + 7)


@pytest.mark.parametrize("format", FORMATS)
def test_an_output_matrix(format):
    same_product(8, 128256, 2048, format, torch.float32, 1)


@pytest.mark.parametrize("M,N,K", [(5, 2048, 4096), (1, 4000, 1800), (16, 1999, 2100), (20, 1000, 8192), (32, 9000, 2048), (1, 512, 16384), (30, 130, 8000),
                                   (33, 1000, 8192), (100, 600, 9001), (128, 2048, 16384), (64, 1, 7937)])
@pytest.mark.parametrize("format", FORMATS)
def test_products_in_parts_of_k(format, M, N, K):
    """Two, four and eight parts of K, whose sums the CTAs of a cluster hand one another."""
    same_product(M, N, K, format, torch.float32, M + N + K)
    same_product(M, N, K, format, torch.bfloat16, M + N + K + 7)


@pytest.mark.parametrize("M,N,K", [(5, 2048, 4096), (20, 500, 8192), (100, 600, 9001), (8, 40000, 256), (1030, 16384, 256), (1500, 2000, 700), (20000, 256, 256)])
@pytest.mark.parametrize("up,down", [(110, -110), (-110, 110), (50, 50), (-55, -55), (-70, -30), (100, -30), (-118, 0), (0, 105)])
@pytest.mark.parametrize("format", FORMATS)
def test_row_scales_at_the_ends_of_the_range(format, M, N, K, up, down):
    """In parts of K and in tiles of two SMs, in some rows beside ordinary ones: sums are whole numbers below 2^24 and the powers of two leave them exact, from
    2^-118 on, to where both are infinite."""
    o = ops()
    x, w = whole(M, K, format, 1, 0), whole(N, K, format, 2, 0)
    ux, uw = torch.zeros(M, device=DEV), torch.zeros(N, device=DEV)
    ux[M // 3:], uw[::2] = up, down
    x, w = x * torch.exp2(ux)[:, None].bfloat16(), w * torch.exp2(uw)[:, None].bfloat16()
    assert x.isfinite().all() and w.isfinite().all()
    want = (x.double() @ w.double().T).float()
    got = o.fp4_gemm(o.fp4_quantize(x, format), o.fp4_quantize(w, format))
    o.check_tc_status()
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows,cols", [(50000, 2048), (3000, 1200), (40000, 250), (40000, 500), (50001, 2047), (1200, 16000), (700, 40000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("format", FORMATS)
def test_many_rows_into_four_bits_and_back(format, dtype, rows, cols):
    """Rows that four bits hold as they are come back as they were; and rows that they do not, sampled, are the nearest."""
    o = ops()
    x = whole(rows, cols, format, rows + cols).to(dtype)
    q = o.fp4_quantize(x, format)
    assert torch.equal(o.fp4_dequantize(q), x.float()) and torch.equal(o.fp4_dequantize(q, torch.bfloat16), x.bfloat16())
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = (torch.randn(rows, cols, generator=g, device=DEV) * torch.exp2(torch.randint(-9, 9, (rows, 1), generator=g, device=DEV).float())).to(dtype)
    q = o.fp4_quantize(x, format)
    at = torch.randint(0, rows, (20,), generator=torch.Generator().manual_seed(cols)).to(DEV)
    at[0], at[1] = 0, rows - 1
    same_values(x[at].cpu(), format, o.fp4_dequantize(q)[at])
    same_values(x[at].cpu(), format, o.fp4_dequantize(q, torch.bfloat16)[at])


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("N,K", [(16384, 700), (9500, 2048), (2000, 1792)])
def test_a_tokens_result_does_not_hang_on_the_others_in_tiles_of_two_sms_either(format, N, K):
    """Where K is not cut into parts every kernel adds along K in the same order."""
    o = ops()
    x, w = rows_like(1301, K, 1).to(DEV), rows_like(N, K, 2).to(DEV)
    qw = o.fp4_quantize(w, format)
    whole_call = o.fp4_gemm(o.fp4_quantize(x, format), qw)
    for n in (1, 16, 17, 33, 100, 129, 257, 600, 1300):
        assert torch.equal(o.fp4_gemm(o.fp4_quantize(x[:n], format), qw), whole_call[:n]), n
    o.check_tc_status()
