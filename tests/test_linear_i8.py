"""The 8-bit dense layers of the box head (ops.quantize_rows_i8, matmul_i8, linear_i8, linear_i8_backward, LinearI8)
against plain 64-bit implementations.

What is exact by construction is compared bit for bit: codes and scales (the nearest whole number of an exact quotient),
and the product (whole-number sums, then the same 64-bit expression and the same roundings as here).  The gradients'
tolerance is the bound of their definition, see `grad_bound`."""
import ctypes

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ------------------------------------------------------------------------------------- plain 64-bit forms (CPU)
def plain_codes(x):
    """x (M,K) CPU -> codes (M,K) float64, scale (M) fp32; the definition, rows with Inf / NaN included."""
    x = x.detach().cpu().double()
    top = x.abs().amax(1)
    good = torch.isfinite(x).all(1) & (top > 0)
    codes = torch.zeros_like(x)
    codes[good] = torch.round(x[good] * 127.0 / top[good, None])  # half to even
    scale = (top / 127.0).float()
    scale[~torch.isfinite(x).all(1)] = float("nan")
    return codes, scale


def plain_product(codes, scale, wcodes, wscale, bias, relu, out_dtype):
    """Sums of products of whole numbers below 2^53 are exact in 64-bit floating point, in any order."""
    z = (codes.double() @ wcodes.double().t()) * scale.double()[:, None] * wscale.double()
    if bias is not None:
        z = z + bias.double()
    if relu:
        z = torch.where(z < 0, torch.zeros_like(z), z)
    return z.float().to(out_dtype)


def plain_grads(grad, y, codes, scale, wcodes, wscale):
    g = grad.double()
    if y is not None:
        g = torch.where(y.double() <= 0, torch.zeros_like(g), g)
    gx = (g * wscale.double()) @ wcodes.double()
    gw = (g * scale.double()[:, None]).t() @ codes.double()
    return g, gx, gw, g.sum(0)


def grad_bound(factors, codes, ref, dtype):
    """factors (R,I), codes (I,C), ref (R,C): each factor is rounded to fp32 (2^-24 of itself) and then to fixed point
    (2^-24 of the row's largest), each error times one code; the result is rounded to fp32 and to `dtype`, half a step
    each (eps / 2 of the value, and half of the smallest subnormal of a 16-bit type)."""
    top = factors.abs().amax(1, keepdim=True)
    fixed = 2 * 2.0 ** -24 * top * codes.abs().sum(0)
    sub = {F16: 2.0 ** -25}.get(dtype, 0.0)
    return fixed + (torch.finfo(dtype).eps / 2 + 2.0 ** -24) * ref.abs() * (1 + 1e-6) + sub


def features(m, k, seed, dtype=F32, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g).relu() * torch.exp(0.7 * torch.randn((1, k), generator=g))
    x[2::7] = 0
    return x.to(dtype).to(dev)


def same_bits(a, b):
    a, b = a.detach().cpu(), b.detach().cpu()
    assert a.shape == b.shape and a.dtype == b.dtype
    nan = torch.isnan(a.float())
    assert torch.equal(nan, torch.isnan(b.float()))
    bad = (a != b) & ~nan
    assert not bad.any(), (int(bad.sum()), a[bad][:4], b[bad][:4])


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    return torch.device("cuda:0")


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_c_entries_refuse_before_any_launch():
    from objectdetection_amd import _lib
    lib = _lib.load()
    p = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused on the host
    null = ctypes.c_void_p(0)

    def refused(rc, word, code=-1):
        assert rc == code and word in lib.frcnn_last_error_string(), (rc, lib.frcnn_last_error_string())

    refused(lib.frcnn_quantize_rows_i8(p, 3, 8, 1, 8, null, p, 16, p, null), b"element type")
    refused(lib.frcnn_quantize_rows_i8(p, 0, 8, 1, 0, null, p, 16, p, null), b"shape")
    refused(lib.frcnn_quantize_rows_i8(p, 0, 8, -1, 8, null, p, 16, p, null), b"shape")
    refused(lib.frcnn_quantize_rows_i8(p, 0, 8, 1, 8, null, p, 7, p, null), b"strides")
    refused(lib.frcnn_quantize_rows_i8(null, 0, 8, 1, 8, null, p, 16, p, null), b"null")
    refused(lib.frcnn_quantize_rows_i8(p, 0, 8, 1, 8, null, ctypes.c_void_p(4104), 16, p, null), b"aligned")
    assert lib.frcnn_quantize_rows_i8(null, 0, 8, 0, 8, null, null, 16, null, null) == 0  # no rows: nothing to do

    def mm(m=4, n=4, k=32, sa=32, sb=32, so=4, a=p, t=0, ws=p, nb=1 << 30):
        return lib.frcnn_matmul_i8(a, sa, p, p, sb, p, null, 0, m, n, k, null, p, t, so, ws, nb, null)
    refused(mm(k=0), b"shape")
    refused(mm(k=131072, sa=131072, sb=131072), b"at most 131071")
    refused(mm(n=0), b"shape")
    refused(mm(sa=-1), b"strides")
    refused(mm(sb=-1), b"strides")
    refused(mm(so=3), b"strides")
    refused(mm(a=null), b"null")
    refused(mm(t=9), b"element type")
    refused(mm(m=40, nb=16), b"workspace", -2)
    refused(mm(m=40, ws=null), b"workspace", -2)
    refused(mm(m=40, ws=ctypes.c_void_p(4096 + 128)), b"aligned")
    refused(mm(m=1 << 22), b"shape")
    refused(lib.frcnn_quantize_rows_i8(p, 0, 8, 1 << 22, 8, null, p, 16, p, null), b"rows")

    def tr(m=40, n=4, k=32, sv=p, sb=1 << 30, wb=1 << 30, x=p):
        return lib.frcnn_linear_i8_train(x, 0, k, p, 0, k, null, 0, m, n, k, p, 0, n, sv, sb, p, wb, null)
    refused(tr(m=0), b"shape")
    refused(tr(k=131072), b"at most 131071")
    refused(tr(x=null), b"null")
    refused(tr(sb=16), b"saved", -2)
    refused(tr(sv=null), b"saved", -2)
    refused(tr(sv=ctypes.c_void_p(4096 + 64)), b"aligned")
    refused(tr(m=4194303), b"M + N")
    refused(lib.frcnn_linear_i8(p, 0, 2048, p, 2048, p, null, 0, 40, 4, 2048, null, p, 0, 4, p, 16, null), b"workspace", -2)
    refused(lib.frcnn_linear_i8(null, 0, 32, p, 32, p, null, 0, 4, 4, 32, null, p, 0, 4, p, 16, null), b"null")
    refused(lib.frcnn_linear_i8(p, 0, 32, p, 32, p, null, 0, 4, 4, 32, null, p, 0, 3, p, 16, null), b"strides")
    refused(lib.frcnn_linear_i8(p, 7, 32, p, 32, p, null, 0, 4, 4, 32, null, p, 0, 4, p, 1 << 30, null), b"element type")

    def bw(m=4, n=4, k=32, a=p, nb=1 << 30):
        return lib.frcnn_linear_i8_backward(p, 0, n, null, 0, a, k, p, p, k, p, m, n, k, p, 0, p, 0, null, p, nb, null)
    refused(bw(m=131072), b"at most 131071")
    refused(bw(k=131072), b"at most 131071")
    refused(bw(a=null), b"null")
    refused(bw(nb=16), b"workspace", -2)
    assert lib.frcnn_linear_i8_workspace_bytes(0, 4, 32) == 0
    assert lib.frcnn_matmul_i8_workspace_bytes(4, 4, 131072) == 0


def test_python_refuses_cpu_tensors():
    from objectdetection_amd import _lib, ops
    x, w, s = torch.zeros(2, 8), torch.zeros((3, 8), dtype=torch.int8), torch.zeros(3)
    with pytest.raises(_lib.FrcnnError):
        ops.quantize_rows_i8(x)
    with pytest.raises(_lib.FrcnnError):
        ops.linear_i8(x, w, s)
    with pytest.raises(_lib.FrcnnError):
        ops.matmul_i8(w[:2], s[:2], w, s)
    with pytest.raises(_lib.FrcnnError):
        ops.LinearI8.apply(x, x, None, False)


@gpu
def test_python_refuses_bad_arguments(dev):
    from objectdetection_amd import ops
    x, w, s = torch.zeros(2, 8, device=dev), torch.zeros((3, 8), dtype=torch.int8, device=dev), torch.zeros(3, device=dev)
    for bad in [lambda: ops.quantize_rows_i8(x[0]), lambda: ops.quantize_rows_i8(x[:, :0]),
                lambda: ops.linear_i8(x, w[:, :7], s), lambda: ops.linear_i8(x, w.float(), s),
                lambda: ops.linear_i8(x, w, s[:2]), lambda: ops.linear_i8(x, w, s, s[:2]),
                lambda: ops.linear_i8(x, w, s, out_dtype=torch.float64), lambda: ops.linear_i8(x, w[:0], s[:0]),
                lambda: ops.linear_i8(x, w, s, n_rows=torch.zeros(2, dtype=torch.int32, device=dev)),
                lambda: ops.matmul_i8(w, s[:2], w, s), lambda: ops.matmul_i8(x, s[:2], w, s),
                lambda: ops.linear_i8_backward(x, None, w[:2], s[:2], w, s),
                lambda: ops.LinearI8.apply(x, w.float()[:, :7], None, False),
                lambda: ops.LinearI8.apply(x.double(), w.float(), None, False)]:
        with pytest.raises(ValueError):
            bad()
    big = torch.zeros((1, ops.I8_MAX_K + 1), device=dev)
    with pytest.raises(ValueError):
        ops.linear_i8(big, big.to(torch.int8), s[:1])


# ---------------------------------------------------------------------------------------------------- quantiser
@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 2), (5, 15), (2, 16), (7, 49), (4, 255), (9, 1024), (3, 1029), (2, 4097),
                                 (3, 12544), (2, 25088), (2, 32769), (1, 70001), (1, 140001)])
def test_quantize_rows(dev, m, k, dtype):
    from objectdetection_amd import ops
    x = features(m, k, 7 * m + k, dtype) * (1 if k % 2 else -1)
    codes, scale = ops.quantize_rows_i8(x.to(dev))
    ref, ref_scale = plain_codes(x)
    assert codes.dtype == torch.int8 and codes.stride(0) % 16 == 0 or m == 1
    assert torch.equal(codes.cpu().double(), ref)
    same_bits(scale, ref_scale)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_quantize_ties_and_extremes(dev, dtype):
    """Halves (x = top (2 n + 1) / 254: exact for these tops), their neighbours one step away, both signs; the largest and
    smallest numbers of a type; zeros; Inf and NaN."""
    from objectdetection_amd import ops
    fin = torch.finfo(dtype)
    rows = []
    for top in (254.0, 127.0, 2.0, 254.0 * 2.0 ** -10):
        h = top * (2 * torch.arange(127, dtype=torch.float64) + 1) / 254
        h = h.to(dtype)
        up, down = (torch.nextafter(h.float(), torch.tensor(t)) for t in (1e9, -1e9))
        row = torch.cat([torch.tensor([top]), h.float(), up, down, -h.float(), -up])
        rows.append(torch.clamp(row, -top, top).to(dtype))
    k = rows[0].numel()
    g = torch.Generator().manual_seed(0)
    for top in (fin.max, fin.tiny, fin.tiny / 2, fin.tiny * fin.eps, fin.tiny * fin.eps * 5, 1e-30 if dtype != F16 else 1e-6):
        r = ((torch.rand((k,), generator=g, dtype=torch.float64) * 2 - 1) * top).to(dtype)
        r[3] = top
        rows.append(r)
    rows.append(torch.zeros(k, dtype=dtype))
    for v in (float("inf"), float("-inf"), float("nan")):
        r = torch.ones(k, dtype=dtype)
        r[k - 1] = v
        rows.append(r)
    x = torch.stack(rows)
    codes, scale = ops.quantize_rows_i8(x.to(dev))
    ref, ref_scale = plain_codes(x)
    bad = (codes.cpu().double() != ref).any(1).nonzero().flatten().tolist()
    assert not bad, (bad, [(codes.cpu()[b].double() - ref[b]).nonzero().flatten()[:5].tolist() for b in bad])
    same_bits(scale, ref_scale)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k", [33001, 65536])
def test_quantize_long_rows(dev, k, dtype):
    """Rows that take two passes: extremes, Inf and NaN in the last element, odd offsets, codes on an odd stride."""
    from objectdetection_amd import _lib, ops
    fin = torch.finfo(dtype)
    base = features(8, k + 3, k, torch.float64)
    base[:, k] = 1.0
    for i, top in enumerate((fin.max, fin.tiny, fin.tiny * fin.eps * 5, 0.0)):
        base[i] *= top / base[i].abs().max()
    base = base.to(dtype)
    base[4, k], base[5, k] = float("inf"), float("nan")
    x = base[:, 1:k + 1]
    ref, ref_scale = plain_codes(x)
    on = base.to(dev)[:, 1:k + 1]
    codes, scale = ops.quantize_rows_i8(on)
    assert torch.equal(codes.cpu().double(), ref)
    same_bits(scale, ref_scale)
    odd = torch.full((8, k + 2 - k % 2), 77, dtype=torch.int8, device=dev)
    P = ctypes.c_void_p
    n = torch.tensor([7], dtype=torch.int32, device=dev)
    assert _lib.load().frcnn_quantize_rows_i8(P(on.data_ptr()), ops._I8_TYPES[dtype], on.stride(0), 8, k, P(n.data_ptr()),
                                              P(odd.data_ptr()), odd.stride(0), P(scale.data_ptr()),
                                              P(torch.cuda.current_stream().cuda_stream)) == 0
    assert torch.equal(odd.cpu()[:7, :k].double(), ref[:7]) and (odd[:, k:] == 77).all() and (odd[7] == 77).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_views_and_counts(dev, dtype):
    from objectdetection_amd import ops
    base = features(20, 333, 5, dtype, dev)
    for x in (base[::3, 5:300], base[:, 1:2], base[4:5, 7:], base.t()[3:9], base[:1].expand(6, 333), base[:, ::2]):
        codes, scale = ops.quantize_rows_i8(x)
        ref, ref_scale = plain_codes(x)
        assert torch.equal(codes.cpu().double(), ref)
        same_bits(scale, ref_scale)
    # rows behind the device-side count are left as they were, padding of a row is zero (C entry: the buffers are ours)
    from objectdetection_amd import _lib
    lib = _lib.load()
    P = ctypes.c_void_p
    for count in (-3, 0, 1, 11, 20, 99):
        codes = torch.full((20, 352), 77, dtype=torch.int8, device=dev)
        scale = torch.full((20,), 5.0, device=dev)
        n = torch.tensor([count], dtype=torch.int32, device=dev)
        rc = lib.frcnn_quantize_rows_i8(P(base.data_ptr()), ops._I8_TYPES[dtype], 333, 20, 333, P(n.data_ptr()),
                                        P(codes.data_ptr()), 352, P(scale.data_ptr()),
                                        P(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        c = max(0, min(20, count))
        ref, ref_scale = plain_codes(base)
        assert torch.equal(codes.cpu()[:c, :333].double(), ref[:c])
        assert (codes[:c, 333:336] == 0).all() and (codes[:c, 336:] == 77).all()
        assert (codes[c:] == 77).all() and (scale[c:] == 5).all()
        same_bits(scale[:c], ref_scale[:c])


# ------------------------------------------------------------------------------------------------------ product
SHAPES = [(1, 1, 1), (1, 3, 15), (2, 5, 16), (3, 7, 17), (1, 64, 128), (16, 16, 64), (17, 33, 129), (31, 65, 255),
          (32, 64, 256), (33, 64, 257), (64, 64, 1024), (65, 65, 1000), (100, 105, 1024), (129, 130, 640), (127, 1, 2048),
          (1, 1024, 12544), (5, 1024, 3136), (300, 21, 12545), (1, 1, 131071), (257, 260, 784), (1000, 105, 100)]


@gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_i8(dev, m, n, k):
    """Bit for bit, at all output types, with and without a bias and a ReLU; the whole range of a byte, -128 included."""
    from objectdetection_amd import ops
    g = torch.Generator().manual_seed(m * 131 + n * 17 + k)
    a = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int32).to(torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8)
    if k == 131071:
        a.fill_(-128), b.fill_(-128)  # the largest sum there is
    sa, sb = torch.rand((m,), generator=g) * 0.1, torch.rand((n,), generator=g) * 0.01
    if m > 2:
        sa[1], sa[2] = 0.0, float("nan")
    bias = torch.randn((n,), generator=g)
    ad, bd, sad, sbd, biasd = (t.to(dev) for t in (a, b, sa, sb, bias))
    for out_dtype, with_bias, relu in [(F32, False, False), (F32, True, True), (BF16, True, False), (F16, False, True)]:
        out = ops.matmul_i8(ad, sad, bd, sbd, biasd if with_bias else None, relu, out_dtype)
        same_bits(out, plain_product(a, sa, b, sb, bias if with_bias else None, relu, out_dtype))


@gpu
@pytest.mark.parametrize("m,n,k", [(13001, 771, 1153), (16300, 1000, 1000), (511, 505, 130001)])
def test_matmul_i8_large_tiles(dev, m, n, k):
    """Sizes that go by 256 x 256 tiles, the last with k split over the chip; rows behind a device-side count."""
    from objectdetection_amd import ops
    g = torch.Generator().manual_seed(k)
    a = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    sa, sb, bias = torch.rand((m,), generator=g) * 0.1, torch.rand((n,), generator=g) * 0.01, torch.randn((n,), generator=g)
    rows = torch.cat([torch.arange(0, m, max(1, m // 300)), torch.tensor([m - 1])])
    ad, bd, sad, sbd, biasd = (t.to(dev) for t in (a, b, sa, sb, bias))
    for out_dtype, relu, count in [(F32, True, None), (BF16, False, None), (F16, True, m - 130), (F32, False, 257)]:
        cnt = torch.tensor([count], dtype=torch.int32, device=dev) if count else None
        out = ops.matmul_i8(ad, sad, bd, sbd, biasd, relu, out_dtype, cnt).cpu()
        at = rows[rows < (count or m)]
        same_bits(out[at], plain_product(a[at], sa[at], b, sb, bias, relu, out_dtype))


@gpu
def test_matmul_i8_views(dev):
    """Rows of any stride and alignment give what contiguous rows give; what lies between them is not read into it."""
    from objectdetection_amd import ops
    g = torch.Generator().manual_seed(3)
    store = torch.randint(-127, 128, (200, 640), generator=g, dtype=torch.int32).to(torch.int8).to(dev)
    s = (torch.rand((200,), generator=g) * 0.1).to(dev)
    for a, b in [(store[:70, :500], store[100:150, 64:564]), (store[:70, 3:500], store[100:150, 64:561]),
                 (store[:70:2, 16:413], store[100:190:3, 5:402]), (store[:6, :33].t()[:, :6], store[100:, :6]),
                 (store[:1, 1:600].expand(9, 599), store[7:8, 16:615])]:
        sa, sb = s[:a.shape[0]], s[100:100 + b.shape[0]]
        out = ops.matmul_i8(a, sa, b, sb, s[:b.shape[0]], True, F32)
        same_bits(out, plain_product(a.cpu(), sa.cpu(), b.cpu(), sb.cpu(), s[:b.shape[0]].cpu(), True, F32))


@gpu
@pytest.mark.parametrize("m,n,k", [(20, 105, 333), (300, 70, 1568), (4, 1024, 6272), (700, 300, 512)])
def test_linear_i8_counts(dev, m, n, k):
    """Rows behind the device-side count are left as they were (C entry: the buffer is ours), also where k is split."""
    from objectdetection_amd import _lib, ops
    lib = _lib.load()
    P = ctypes.c_void_p
    x = features(m, k, 11)
    w = torch.randn((n, k), generator=torch.Generator().manual_seed(1))
    wc, ws = plain_codes(w)
    q, s = plain_codes(x)
    ref = plain_product(q, s, wc, ws, None, False, F32)
    xd, wd, wsd = x.to(dev), wc.to(torch.int8).to(dev), ws.to(dev)
    nbytes = lib.frcnn_linear_i8_workspace_bytes(m, n, k)
    work = torch.randint(0, 255, (nbytes,), dtype=torch.uint8, device=dev)
    for count in (-1, 0, 1, m // 2 + 1, m, m + 50):
        out = torch.full((m, n + 3), 5.0, device=dev)
        cnt = torch.tensor([count], dtype=torch.int32, device=dev)
        rc = lib.frcnn_linear_i8(P(xd.data_ptr()), 0, k, P(wd.data_ptr()), k, P(wsd.data_ptr()), P(0), 0, m, n, k,
                                 P(cnt.data_ptr()), P(out.data_ptr()), 0, n + 3, P(work.data_ptr()), nbytes,
                                 P(torch.cuda.current_stream().cuda_stream))
        assert rc == 0, lib.frcnn_last_error_string()
        c = max(0, min(m, count))
        same_bits(out[:c, :n], ref[:c])
        assert (out[c:] == 5).all() and (out[:, n:] == 5).all()
    out = ops.linear_i8(xd, wd, wsd, n_rows=torch.tensor([m // 2], device=dev))
    same_bits(out[:m // 2], ref[:m // 2])
    assert ops.linear_i8(xd[:0], wd, wsd).shape == (0, n)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", [(1, 1024, 1024), (37, 105, 1029), (2, 1, 1), (513, 129, 2401)])
def test_linear_i8(dev, m, n, k, dtype):
    """From float rows to float rows; a row of zeros gives the bias, a row with an Inf or a NaN gives NaN."""
    from objectdetection_amd import ops
    x = features(m, k, 13, dtype)
    if m > 30:
        x[4, k // 2], x[9, 0] = float("inf"), float("nan")
    g = torch.Generator().manual_seed(2)
    w, bias = torch.randn((n, k), generator=g) * 0.05, torch.randn((n,), generator=g)
    wc, ws = ops.quantize_rows_i8(w.to(dev))
    out = ops.linear_i8(x.to(dev), wc, ws, bias.to(dev), relu=True)
    assert out.dtype == dtype
    q, s = plain_codes(x)
    p, t = plain_codes(w)
    ref = plain_product(q, s, p, t, bias, True, dtype)
    same_bits(out, ref)
    if m > 30:
        assert torch.isnan(out[4]).all() and torch.isnan(out[9]).all() and not torch.isnan(out[5]).any()


# The three forms (a few rows; short rows, 16 and 64 a workgroup; quantiser and tiles) at the edges between them: rows,
# channels and lengths beside multiples of 16, 64 and 128, the last weight in the middle of a 16-byte load.
FORMS = [(1, 1, 15), (2, 7, 17), (4, 5, 4099), (3, 4, 32768), (4, 9, 32769), (5, 3, 16), (3, 1, 16), (16, 16, 31), (17, 15, 33),
         (15, 129, 63), (64, 2, 65), (65, 105, 127), (100, 257, 1023), (63, 300, 1024), (33, 40, 1025), (130, 128, 1009),
         (20000, 21, 49), (16500, 130, 48), (17000, 128, 1000), (9000, 300, 80), (5, 513, 1007), (300, 1, 77)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_linear_i8_forms(dev, m, n, k, dtype):
    from objectdetection_amd import ops
    fin = torch.finfo(dtype)
    x = features(m, k, 3 * m + k, dtype)
    x[:, 1::2] *= -1
    # rows at the ends of the type, of ties, with an Inf and a NaN, spread over the workgroups
    for i, r in enumerate(range(0, m, max(1, m // 9))):
        if i % 9 == 1:
            x[r] = (x[r].double() / max(float(x[r].abs().max()), 1e-9) * fin.max).to(dtype)
        elif i % 9 == 2:
            x[r] = (x[r].double() * fin.tiny * 0.3).to(dtype)
        elif i % 9 == 3:
            x[r] = (torch.arange(k) % 255 - 127).double().mul(0.5).to(dtype)
            x[r, k // 3] = 127.0
        elif i % 9 == 4:
            x[r, k - 1] = float("inf")
        elif i % 9 == 5:
            x[r, 0] = float("nan")
        elif i % 9 == 6:
            x[r] = 0
    g = torch.Generator().manual_seed(k)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8)
    ws, bias = torch.rand((n,), generator=g) * 0.01, torch.randn((n,), generator=g)
    out = ops.linear_i8(x.to(dev), w.to(dev), ws.to(dev), bias.to(dev), True, F32)
    q, s = plain_codes(x)
    same_bits(out, plain_product(q, s, w, ws, bias, True, F32))
    # weight rows on a stride of their own behind an odd offset, rows of x on another, no bias, the type's own output
    store = torch.zeros((n, k + 13), dtype=torch.int8, device=dev)
    store[:, 5:5 + k] = w.to(dev)
    wide = torch.full((m, k + 3), float("nan"), dtype=dtype, device=dev)
    wide[:, 1:1 + k] = x.to(dev)
    out = ops.linear_i8(wide[:, 1:1 + k], store[:, 5:5 + k], ws.to(dev))
    same_bits(out, plain_product(q, s, w, ws, None, False, dtype))


# ---------------------------------------------------------------------------------------------------- gradients
@gpu
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5, 33), (3, 130, 17), (63, 65, 127), (130, 105, 260), (257, 21, 1029),
                                   (64, 1024, 196), (700, 3, 50)])
def test_gradients_against_the_formulas(dev, m, n, k, dtype, wdtype, relu):
    from objectdetection_amd import ops
    g = torch.Generator().manual_seed(m + 3 * n + 5 * k)
    x = features(m, k, 17, dtype, dev).requires_grad_()
    w = (torch.randn((n, k), generator=g) * 0.05).to(wdtype).to(dev).requires_grad_()
    bias = torch.randn((n,), generator=g).to(dev).requires_grad_()
    # heavy-tailed, as losses leave them: a few rows thousands of times the others
    grad = (torch.randn((m, n), generator=g) * torch.exp(2 * torch.randn((m, 1), generator=g)) * 0.05).to(dtype).to(dev)
    y = ops.LinearI8.apply(x, w, bias, relu)
    q, s = plain_codes(x)
    p, t = plain_codes(w)
    same_bits(y, plain_product(q, s, p, t, bias.detach().cpu(), relu, dtype))
    gx, gw, gb = torch.autograd.grad(y, (x, w, bias), grad)
    assert gx.dtype == dtype and gw.dtype == wdtype and gb.dtype == F32
    gm, rx, rw, rb = plain_grads(grad.cpu(), y.detach().cpu() if relu else None, q, s, p, t)
    fx, fw = gm * t.double(), (gm * s.double()[:, None]).t()
    assert ((gx.cpu().double() - rx).abs() <= grad_bound(fx, p, rx, dtype)).all()
    assert ((gw.cpu().double() - rw).abs() <= grad_bound(fw, q, rw, wdtype)).all()
    # an fp32 sum in some order: each of its m - 1 additions rounds by 2^-24 of at most the sum of magnitudes
    assert ((gb.cpu().double() - rb).abs() <= (m + 1) * 2.0 ** -24 * gm.abs().sum(0) + 1e-45).all()
    # the same bits again, and for each gradient alone
    again = torch.autograd.grad(ops.LinearI8.apply(x, w, bias, relu), (x, w, bias), grad)
    for u, v in zip(again, (gx, gw, gb)):
        same_bits(u, v)
    for i, leaf in enumerate((x, w, bias)):
        leaves = [v.detach() for v in (x, w, bias)]
        leaves[i] = leaf
        same_bits(torch.autograd.grad(ops.LinearI8.apply(*leaves, relu), leaf, grad)[0], (gx, gw, gb)[i])


@gpu
@pytest.mark.parametrize("m,n,k", [(2049, 40, 70), (5003, 33, 130), (70, 2500, 65), (40, 4101, 20), (2300, 2200, 64)])
def test_gradients_of_long_sums(dev, m, n, k):
    """Sums over many rows or channels: in one piece, and split over workgroups and joined."""
    test_gradients_against_the_formulas(dev, m, n, k, F32, F32, True)
    test_gradients_against_the_formulas(dev, m, n, k, BF16, F32, False)


@gpu
def test_gradients_against_differences(dev):
    """The straight-through gradient is that of f = sum(grad * relu(X W^T + b)) at the dequantised X, W: central
    differences of f in 64 bits, along random directions.  f is piecewise linear in each argument, so away from a kink a
    central difference is exact up to 64-bit rounding; h keeps every z on its side."""
    from objectdetection_amd import ops
    m, n, k = 40, 30, 64
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn((m, k), generator=g).to(dev).requires_grad_(), torch.randn((n, k), generator=g).to(dev).requires_grad_()
    b = torch.randn((n,), generator=g).to(dev).requires_grad_()
    grad = torch.randn((m, n), generator=g)
    got = torch.autograd.grad(ops.LinearI8.apply(x, w, b, True), (x, w, b), grad.to(dev))
    q, s = plain_codes(x)
    p, t = plain_codes(w)
    at = [q * s.double()[:, None], p * t.double()[:, None], b.detach().cpu().double()]

    def f(v):
        return float((grad.double() * (v[0] @ v[1].t() + v[2]).clamp(min=0)).sum())
    z = at[0] @ at[1].t() + at[2]
    for i in range(3):
        d = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        h = 1e-7
        plus, minus = [list(at) for _ in range(2)]
        plus[i], minus[i] = at[i] + h * d, at[i] - h * d
        zp = plus[0] @ plus[1].t() + plus[2]
        assert torch.equal(zp > 0, z > 0)
        slope = (f(plus) - f(minus)) / (2 * h)
        mine = float((got[i].cpu().double() * d).sum())
        # 2^-53 of f's magnitude over 2 h, and the gradients' own bound (2^-23 relative, generously 1e-6)
        scale = float((got[i].cpu().double().abs() * d.abs()).sum())
        total = float((grad.double().abs() * z.abs()).sum())
        assert abs(slope - mine) <= 1e-6 * scale + 64 * 2.0 ** -53 * total / h


@gpu
def test_gradients_of_odd_inputs(dev):
    """Broadcast and strided gradients, no rows at all, rows that get no gradient, Inf in a gradient, a second call of
    backward refused."""
    from objectdetection_amd import ops
    x = features(20, 50, 3).to(dev).requires_grad_()
    w = torch.randn((6, 50), generator=torch.Generator().manual_seed(1)).to(dev).requires_grad_()
    q, s = plain_codes(x)
    p, t = plain_codes(w)
    for make in (lambda y: y.sum(), lambda y: (y[:, 2:5] * 3).sum(), lambda y: y.t().contiguous().sum(), lambda y: y[::4].sum()):
        y = ops.LinearI8.apply(x, w, None, False)
        grad, = torch.autograd.grad(make(y), y, retain_graph=True)
        gx, gw = torch.autograd.grad(make(y), (x, w))
        gm, rx, rw, _ = plain_grads(grad.cpu(), None, q, s, p, t)
        assert ((gx.cpu().double() - rx).abs() <= grad_bound(gm * t.double(), p, rx, F32)).all()
        assert ((gw.cpu().double() - rw).abs() <= grad_bound((gm * s.double()[:, None]).t(), q, rw, F32)).all()
    none = ops.LinearI8.apply(x[:0], w, None, True)
    gx, gw = torch.autograd.grad(none.sum(), (x, w))
    assert none.shape == (0, 6) and not gx.any() and not gw.any()
    grad = torch.ones((20, 6), device=dev)
    grad[3, 1] = float("inf")
    gx, gw = torch.autograd.grad(ops.LinearI8.apply(x, w, None, False), (x, w), grad)
    bad_x, bad_w = torch.isnan(gx).all(1), torch.isnan(gw).all(1)
    assert bad_x[3] and bad_w[1] and int(bad_x.sum()) == 1 and int(bad_w.sum()) == 1
    assert torch.isfinite(gx[~bad_x]).all() and torch.isfinite(gw[~bad_w]).all()
    y = ops.LinearI8.apply(x, w, None, True)
    first, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


# ------------------------------------------------------------------------------------------- streams and graphs
@gpu
def test_other_stream_and_captured_replays(dev):
    """On a side stream, and captured: replayed several times on new inputs with eager work between, each against the
    eager result."""
    from objectdetection_amd import ops
    x = features(60, 700, 1).to(dev)
    w = torch.randn((40, 700), generator=torch.Generator().manual_seed(5)).to(dev)
    grad = torch.randn((60, 40), generator=torch.Generator().manual_seed(6)).to(dev)
    wc, ws = ops.quantize_rows_i8(w)

    def step():
        y = ops.linear_i8(x, wc, ws, None, True)
        c, s = ops.quantize_rows_i8(x)
        return (y,) + ops.linear_i8_backward(grad, y, c, s, wc, ws)
    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    for u, v in zip(other, eager):
        same_bits(u, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(features(60, 700, 20 + i).to(dev) * (i + 1))
        grad.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for u, v in zip(got, step()):
            same_bits(u, v)


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 300, 2100), (99, 1024, 4100), (700, 400, 2048), (2000, 520, 1030)])
def test_forms_captured_and_on_two_streams(dev, m, n, k):
    """One launch, short rows and tiles with a split k: two streams work at once on inputs of their own, and two captured
    calls are replayed in turn on new inputs, each against the eager result."""
    from objectdetection_amd import ops
    wc, ws = ops.quantize_rows_i8(torch.randn((n, k), generator=torch.Generator().manual_seed(9)).to(dev))
    xs = [features(m, k, 30 + i).to(dev) for i in range(2)]
    eager = [ops.linear_i8(x, wc, ws, None, True) for x in xs]
    streams = [torch.cuda.Stream(device=dev) for _ in xs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.linear_i8(xs[i], wc, ws, None, True))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            same_bits(y, eager[i])
    graphs, held = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(ops.linear_i8(x, wc, ws, None, True))
        graphs.append(graph)
    for r in range(3):
        for i, x in enumerate(xs):
            x.copy_(features(m, k, 40 + 2 * r + i).to(dev))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i, x in enumerate(xs):
            same_bits(held[i], ops.linear_i8(x, wc, ws, None, True))


@gpu
def test_captured_training_step(dev):
    """Forward and backward of LinearI8 recorded into one graph and replayed on new inputs and weights."""
    from objectdetection_amd import ops
    x = features(130, 300, 3).to(dev).requires_grad_()
    w = torch.randn((40, 300), generator=torch.Generator().manual_seed(5)).to(dev).requires_grad_()
    b = torch.randn((40,), generator=torch.Generator().manual_seed(7)).to(dev).requires_grad_()
    up = torch.randn((130, 40), generator=torch.Generator().manual_seed(6)).to(dev)

    def step():
        y = ops.LinearI8.apply(x, w, b, True)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), up)
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(features(130, 300, 50 + i).to(dev))
            w.mul_(0.5)
            up.neg_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for u, v in zip(got, step()):
            same_bits(u, v)


# ------------------------------------------------------------------------------------------------- the box head
def _float_head(dev, in_channels=3 * 49, rep=70, classes=5, int8=False):
    from objectdetection_amd.ROIHead import FasterRCNNPredictor, TwoMLPHead
    torch.manual_seed(11)
    return (TwoMLPHead(in_channels, rep, int8=int8).to(dev), FasterRCNNPredictor(rep, classes, int8=int8).to(dev))


def _plain_layer(x, weight, bias, relu):
    q, s = plain_codes(x)
    p, t = plain_codes(weight)
    return plain_product(q, s, p, t, bias.detach().cpu(), relu, F32)


def _plain_head(x, head, pred):
    """The served box head in 64 bits, layer by layer on the CPU."""
    y = _plain_layer(x.flatten(1).cpu(), head.fc1.weight, head.fc1.bias, True)
    y = _plain_layer(y, head.fc2.weight, head.fc2.bias, True)
    return _plain_layer(y, pred.cls_score.weight, pred.cls_score.bias, False), \
        _plain_layer(y, pred.bbox_pred.weight, pred.bbox_pred.bias, False)


@gpu
def test_served_box_head_behind_the_padded_pooling(dev):
    """pool.forward_padded -> Int8TwoMLPHead -> Int8FasterRCNNPredictor with the device-side row count: the pooled rows
    behind it hold NaN here, and the valid rows come out as from the unpadded features."""
    from objectdetection_amd.ROIHead import Int8FasterRCNNPredictor, Int8TwoMLPHead, ROIPooling
    head, pred = _float_head(dev)
    served, served_pred = Int8TwoMLPHead.from_float(head).eval(), Int8FasterRCNNPredictor.from_float(pred).eval()
    g = torch.Generator().manual_seed(3)
    feat = torch.randn((2, 3, 20, 30), generator=g).relu().to(dev)
    xy = torch.rand((2, 40, 2), generator=g) * 200
    props = torch.cat([xy, xy + 20 + torch.rand((2, 40, 2), generator=g) * 100], 2).to(dev)
    count = torch.tensor([40, 23], dtype=torch.int32, device=dev)
    props[1, 23:] = 0
    pool = ROIPooling(['1'], [7, 7], 2)
    feats, total = pool.forward_padded({'1': feat}, props, count, [(320, 480)])
    assert int(total) == 63
    feats[63:] = float("nan")
    cls, reg = served_pred(served(feats, total), total)
    ref_cls, ref_reg = _plain_head(feats[:63], head, pred)
    same_bits(cls[:63], ref_cls)
    same_bits(reg[:63], ref_reg)
    # and without a count, on the valid rows alone
    cls, reg = served_pred(served(feats[:63]))
    same_bits(cls, ref_cls)
    same_bits(reg, ref_reg)


@gpu
def test_roi_head_serves_and_trains_through_int8(dev):
    """ROIHead with the 8-bit layers: detections are those of the plain layers put in their place; its training branch
    leaves the gradients that the chain of single calls gives, bit for bit, on the weights and on the feature maps."""
    from objectdetection_amd import ops
    from objectdetection_amd.ROIHead import Int8FasterRCNNPredictor, Int8TwoMLPHead, ROIHead, ROIPooling
    g = torch.Generator().manual_seed(8)
    xy = torch.rand((2, 60, 2), generator=g) * 150
    boxes = torch.cat([xy, xy + 20 + torch.rand((2, 60, 2), generator=g) * 90], 2).to(dev)
    props = [boxes[0], boxes[1, :35]]
    targets = [{'size': [3.0, 281, 500], 'class': [1.0, 2.0], 'box': [[104, 78, 175, 183], [33, 88, 197, 123]]},
               {'size': [3.0, 500.0, 375.0], 'class': [2.0], 'box': [[104, 78, 205, 183]]}]
    head, pred = _float_head(dev)
    with torch.no_grad():
        pred.cls_score.weight.mul_(20)  # scores apart from each other
    base = dict(pos_threshold=0.3, neg_threshold=0.3, num_sample=64, pos_fraction=0.25,
                regression_weights=[10., 10., 5., 5.], score_thresh=0.05, proposal_min_size=1e-3, nms_threshold=0.5,
                num_post_nms=50, roi_pooling=ROIPooling(['1', '2'], [7, 7], 2))
    feats = [torch.randn((2, 3, 128, 128), generator=g).relu().to(dev), torch.randn((2, 3, 64, 64), generator=g).relu().to(dev)]

    class Plain(torch.nn.Module):
        def forward(self, x):
            return x.flatten(1)

    class PlainPredictor(torch.nn.Module):
        def forward(self, x):
            return tuple(t.to(dev) for t in _plain_head(x, head, pred))
    args = (props, feats, (2, 256, 256), targets, [(250, 226), (256, 240)])
    with torch.no_grad():
        got, _ = ROIHead(dict(base, mlp_head=Int8TwoMLPHead.from_float(head),
                              predictor=Int8FasterRCNNPredictor.from_float(pred)))(*args)
        ref, _ = ROIHead(dict(base, mlp_head=Plain(), predictor=PlainPredictor()))(*args)
    assert sum(len(r['score']) for r in ref) > 10
    for a, b in zip(got, ref):
        for key in ('proposal', 'score', 'label'):
            assert torch.equal(a[key], b[key])

    head, pred = _float_head(dev, int8=True)
    maps = [f.clone().requires_grad_() for f in feats]
    trained = ROIHead(dict(base, mlp_head=head, predictor=pred, force_eval=False)).train()
    torch.manual_seed(4)
    _, loss = trained(props, maps, (2, 256, 256), targets, [(250, 226), (256, 240)])
    (loss["cls_loss"] + loss["reg_loss"]).backward()
    # the same step by single calls
    sampled = trained.last_sampled
    again = [f.clone().requires_grad_() for f in feats]
    pooled = trained.roi_pooling({'1': again[0], '2': again[1]}, [s["proposal"] for s in sampled], [(256, 256)])
    x = pooled.flatten(1)
    w3 = torch.cat([pred.cls_score.weight, pred.bbox_pred.weight]).detach()
    b3 = torch.cat([pred.cls_score.bias, pred.bbox_pred.bias]).detach()
    layers, y = [], x.detach()
    for w, b, relu in ((head.fc1.weight, head.fc1.bias, True), (head.fc2.weight, head.fc2.bias, True), (w3, b3, False)):
        c, s = ops.quantize_rows_i8(y)
        p, t = ops.quantize_rows_i8(w)
        y = ops.matmul_i8(c, s, p, t, b, relu)
        layers.append((c, s, p, t, y if relu else None))
    n = pred.cls_score.out_features
    _, gl, gp = ops.roi_loss(y[:, :n], y[:, n:], torch.cat([s["cls_label"] for s in sampled]),
                             torch.cat([s["reg_label"] for s in sampled]))
    grad, grads = torch.cat([gl, gp.reshape(gl.shape[0], -1)], 1), []
    for c, s, p, t, out in reversed(layers):
        grad, gw, gb = ops.linear_i8_backward(grad, out, c, s, p, t)
        grads.append((gw, gb))
    same_bits(grads[2][0], head.fc1.weight.grad)
    same_bits(grads[2][1], head.fc1.bias.grad)
    same_bits(grads[1][0], head.fc2.weight.grad)
    same_bits(grads[0][0], torch.cat([pred.cls_score.weight.grad, pred.bbox_pred.weight.grad]))
    same_bits(grads[0][1], torch.cat([pred.cls_score.bias.grad, pred.bbox_pred.bias.grad]))
    x.backward(grad)
    for a, b in zip(maps, again):
        # RoIAlign's backward adds with atomics for maps of this size: the order of its sums is not fixed
        torch.testing.assert_close(a.grad, b.grad, rtol=1e-4, atol=1e-6 * float(b.grad.abs().max()))
    assert head.fc1.weight.grad.abs().sum() > 0 and maps[0].grad.abs().sum() > 0


def test_scales_stay_in_32_bits_and_old_modules_load():
    from objectdetection_amd.ROIHead import FasterRCNNPredictor, Int8Linear, Int8TwoMLPHead, TwoMLPHead
    scale = torch.full((4,), 1.2345678e-7)
    for cast in (lambda m: m.half(), lambda m: m.to(BF16), lambda m: m.double(), lambda m: m.float()):
        layer = Int8Linear(8, 4)
        layer.scale.copy_(scale)
        layer = cast(layer)
        assert layer.scale.dtype == layer.bias.dtype == F32 and layer.codes.dtype == torch.int8
        assert torch.equal(layer.scale, scale)
    assert Int8Linear(8, 4, bias=False).half().bias is None
    head = Int8TwoMLPHead(8, 4).half()
    assert head.fc1.scale.dtype == F32 and set(dict(head.named_buffers())) == set(head.state_dict())
    for old in (TwoMLPHead(8, 4), FasterRCNNPredictor(4, 3)):  # as restored from before the choice
        del old.__dict__["int8"]
        old(torch.zeros((2, old.fc1.in_features if hasattr(old, "fc1") else 4)))


@gpu
def test_int8_modules_keep_and_refuse(dev):
    from objectdetection_amd import _lib
    from objectdetection_amd.ROIHead import Int8FasterRCNNPredictor, Int8Linear, Int8TwoMLPHead, TwoMLPHead
    head, pred = _float_head(dev)
    served = Int8TwoMLPHead.from_float(head)
    other = Int8TwoMLPHead(3 * 49, 70).to(dev)
    other.load_state_dict(served.state_dict())
    x = features(9, 3 * 49, 2).to(dev)
    same_bits(other(x), served(x))
    assert set(served.state_dict()) == {"fc1.codes", "fc1.scale", "fc1.bias", "fc2.codes", "fc2.scale", "fc2.bias"}
    assert not list(served.parameters())
    loaded = Int8FasterRCNNPredictor(70, 5).to(dev)
    loaded.load_state_dict(Int8FasterRCNNPredictor.from_float(pred).state_dict())
    assert [t.shape for t in loaded(served(x))] == [(9, 5), (9, 20)]
    bare = Int8Linear.from_float(head.fc2.weight)  # no bias, no ReLU, 16-bit output
    y = bare(x[:, :70], out_dtype=BF16)
    assert y.dtype == BF16 and (y < 0).any() and bare.bias is None
    with pytest.raises(RuntimeError):
        served.train()(x.requires_grad_())
    served.eval()(x)  # serving: the result is detached
    with torch.no_grad():
        served.train()(x)
    with pytest.raises(_lib.FrcnnError):
        Int8TwoMLPHead.from_float(TwoMLPHead(8, 8))  # weights on the CPU
    # same parameters, trained in 8 bits or not
    assert set(TwoMLPHead(8, 8, int8=True).state_dict()) == set(TwoMLPHead(8, 8).state_dict())
