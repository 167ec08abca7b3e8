"""The 8-bit dense layers of the box head beyond the sizes and the values of tests/test_linear_i8.py: what 32 bits of an index
cannot hold, signs that hang on the last bit, gradients of very different sizes, modules as a user wires them up."""
import ctypes

import pytest
import torch

from .test_linear_i8 import BF16, F16, F32, dev, features, gpu, plain_codes, plain_grads, plain_product, same_bits  # noqa: F401
from .test_linear_i8 import test_gradients_against_the_formulas as _against_the_formulas


# ------------------------------------------------------------------------------------------------ sizes past 32 bits
def test_rows_too_long_for_an_index_are_refused():
    """Column indices are 32-bit numbers: a row that they cannot step past is refused before any launch."""
    from objectdetection_amd import _lib, ops
    lib = _lib.load()
    p, null = ctypes.c_void_p(4096), ctypes.c_void_p(0)  # never dereferenced
    for k in ((1 << 30) + 1, (1 << 31) - 20000, (1 << 31) - 1):
        assert lib.frcnn_quantize_rows_i8(p, 1, k, 1, k, null, p, k + 1 | 1, p, null) == -1
        assert b"shape" in lib.frcnn_last_error_string()
    assert lib.frcnn_quantize_rows_i8(p, 1, 1 << 30, 0, 1 << 30, null, p, 1 << 30, p, null) == 0  # no rows: nothing to do
    for sizes in ((1 << 22, 1, 8), (1 << 32, 1, 8), (1, (1 << 32) + 3, 8), (1, 1, 1 << 17), (1, 1, (1 << 32) + 5)):
        with pytest.raises(ValueError):
            ops._i8_sizes("sizes", *sizes)
    ops._i8_sizes("sizes", ops.I8_MAX_ROWS, ops.I8_MAX_ROWS, ops.I8_MAX_K)


@gpu
def test_python_refuses_sizes_past_32_bits(dev):
    """Views of a few bytes with more rows or columns than a C int holds: refused, not cut to their low 32 bits."""
    from objectdetection_amd import ops
    x = torch.ones((1, 8), device=dev, dtype=BF16)
    codes, scale = ops.quantize_rows_i8(x)
    many, long = x.expand((1 << 32) + 1, 8), x[:, :1].expand(1, (1 << 32) + 5)
    many_codes, many_scale = codes.expand((1 << 32) + 1, 8), scale.expand((1 << 32) + 1)
    for bad in (lambda: ops.quantize_rows_i8(many), lambda: ops.quantize_rows_i8(long),
                lambda: ops.quantize_rows_i8(x.expand(1 << 22, 8)), lambda: ops.linear_i8(many, codes, scale),
                lambda: ops.linear_i8(x, many_codes, many_scale), lambda: ops.matmul_i8(many_codes, many_scale, codes, scale),
                lambda: ops.linear_i8(long, codes[:, :1].expand(1, (1 << 32) + 5), scale),
                lambda: ops.LinearI8.apply(many, x, None, False), lambda: ops.LinearI8.apply(x, many, None, False)):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------------------- gradients whose factors differ widely in size
def float_bound(factors, codes, ref, dtype):
    """factors (R,I), codes (I,C), ref (R,C).  A factor is held to 2^-23 of itself, or 2^-50 of its row's largest; its product
    with a code is exact; the I products of an output are added in fp32, each addition off by at most one step, 2^-23, of
    what has been added, which is at most the sum of magnitudes (the second pieces' sum, 2^-10 of that, likewise); the result
    is rounded to fp32 and to `dtype`, half a step of each, and half of the smallest subnormal number."""
    inner = codes.shape[0]
    top = factors.abs().amax(1, keepdim=True)
    held = (1 + inner * (1 + 2.0 ** -10)) * 2.0 ** -23 * (factors.abs() @ codes.abs()) + 2.0 ** -50 * top * codes.abs().sum(0)
    sub = {F16: 2.0 ** -25, BF16: 2.0 ** -134}.get(dtype, 0.0) + 2.0 ** -150
    return held + (torch.finfo(dtype).eps / 2 + 2.0 ** -24) * (ref.abs() + held) + sub


def _skewed(kind, m, n, g):
    if kind == "confident":  # cross-entropy of a classifier that is sure, and mostly right
        logits = 12 * torch.randn((m, n), generator=g)
        label = torch.where(torch.rand((m,), generator=g) < 0.98, logits.argmax(1), torch.randint(0, n, (m,), generator=g))
        logits[torch.arange(m), label] += 12
        p = torch.softmax(logits, 1)
        p[torch.arange(m), label] -= 1
        return p / m
    grad = 0.05 * torch.randn((m, n), generator=g)
    if kind == "tiny":  # the factors are subnormal numbers of fp32
        return grad * 1e-37
    grad[m // 3] *= kind  # one row far above the others
    return grad


@gpu
@pytest.mark.parametrize("kind", ["confident", 1e6, 1e9, 1e15, "tiny"])
@pytest.mark.parametrize("m,n,k,relu", [(2048, 105, 300, False), (130, 37, 64, True), (70, 2500, 65, False), (5003, 33, 130, True)])
def test_gradients_of_factors_far_apart(dev, m, n, k, relu, kind):
    """Against the formulas, each output by the magnitudes of its OWN terms: features are sparse, so that many outputs have
    nothing of the row's or the column's largest factor in them."""
    from objectdetection_amd import ops
    g = torch.Generator().manual_seed(m + n)
    x = features(m, k, 23) * (torch.rand((m, k), generator=g) < 0.1)
    w = torch.randn((n, k), generator=g) * 0.05 * (torch.rand((n, k), generator=g) < 0.2)
    grad = _skewed(kind, m, n, g)
    leaves = [t.to(dev).requires_grad_() for t in (x, w)]
    y = ops.LinearI8.apply(leaves[0], leaves[1], None, relu)
    gx, gw = torch.autograd.grad(y, leaves, grad.to(dev))
    (q, s), (p, t) = plain_codes(x), plain_codes(w)
    gm, rx, rw, _ = plain_grads(grad, y.detach().cpu() if relu else None, q, s, p, t)
    fx, fw = gm * t.double(), (gm * s.double()[:, None]).t()
    for got, f, c, ref in ((gx, fx, p, rx), (gw, fw, q, rw)):
        bad = (got.cpu().double() - ref).abs() > float_bound(f, c, ref, F32)
        assert not bad.any(), (int(bad.sum()), bad.numel(), got.cpu()[bad][:3], ref[bad][:3])


@gpu
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32)])
@pytest.mark.parametrize("m,n,k", [(257, 1030, 12545), (2100, 130, 7000)])
def test_gradients_by_large_tiles(dev, m, n, k, dtype, wdtype):
    """Products with enough tiles of 128 x 256 to fill the chip, none of their sides a multiple of a tile's."""
    _against_the_formulas(dev, m, n, k, dtype, wdtype, True)


# ------------------------------------------------------------------------------------ signs that hang on the last bit
def _row_with_sum(total, k):
    """Bytes a, b (k) with sum a b = total (>= 0)."""
    a, b = torch.zeros(k, dtype=torch.int64), torch.zeros(k, dtype=torch.int64)
    full, rest = divmod(total, 127 * 127)
    assert full + 2 <= k
    a[:full] = b[:full] = 127
    a[full], b[full] = 127, rest // 127
    a[full + 1], b[full + 1] = 1, rest % 127
    assert int((a * b).sum()) == total
    return a.to(torch.int8), b.to(torch.int8)


@gpu
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("m", [2, 40])
def test_sign_of_a_sum_that_53_bits_do_not_hold(dev, m, sign):
    """sum * a_scale needs 55 bits and the bias cancels all but its last: what is left is one unit, to which the ReLU's sign
    and the result's value both hang."""
    from objectdetection_amd import ops
    k = 131071
    scale = next(v for v in range((1 << 24) - 1, 1 << 23, -2)  # an odd 24-bit number, times its inverse modulo 2^31
                 if 2060000000 < pow(v, -1, 1 << 31) * sign % (1 << 31) < 2110000000)
    total = pow(scale, -1, 1 << 31) * sign % (1 << 31)
    left = total * scale - sign
    assert left % (1 << 31) == 0 and left >> 31 < 1 << 24 and (total * scale).bit_length() == 55
    a, b = _row_with_sum(total, k)
    codes = a.repeat(m, 1).to(dev)
    unit = 2.0 ** -20
    out = ops.matmul_i8(codes, torch.full((m,), float(scale), device=dev), b[None].to(dev), torch.tensor([unit], device=dev),
                        torch.tensor([-float(left) * unit], device=dev), False)
    assert (out == sign * unit).all(), out[:2]
    out = ops.matmul_i8(codes, torch.full((m,), float(scale), device=dev), b[None].to(dev), torch.tensor([unit], device=dev),
                        torch.tensor([-float(left) * unit], device=dev), True)
    assert (out == max(sign, 0) * unit).all(), out[:2]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", [(3, 40, 100), (60, 70, 300), (99, 64, 4100), (600, 520, 1100), (40, 33, 33001)])
def test_relu_lets_gradients_through_where_the_sum_is_positive(dev, m, n, k, dtype):
    """Outputs around the border where their type rounds to zero: the gate is the sum's sign, not the rounded output's.  The
    output itself stays the rounded one."""
    from objectdetection_amd import ops
    g = torch.Generator().manual_seed(k)
    low = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}[dtype]  # rounds to zero, and what is above does not
    x = features(m, k, 31, torch.float64) * (2.0 ** -70 if dtype != F16 else 1.0)
    x = x.to(dtype)
    w = torch.randn((n, k), generator=g)
    w *= low / float((x.double() @ w.double().t()).abs().median())
    grad = torch.randn((m, n), generator=g).to(dtype)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, torch.zeros(n))]
    y = ops.LinearI8.apply(*leaves, True)
    gx, gw, gb = torch.autograd.grad(y, leaves, grad.to(dev))
    (q, s), (p, t) = plain_codes(x), plain_codes(w)
    same_bits(y, plain_product(q, s, p, t, None, True, dtype))
    z = (q @ p.t()) * s.double()[:, None] * t.double()
    assert ((z > 0) & (y.cpu() == 0)).sum() > m * n / 20 and (y > 0).sum() > m * n / 20
    gm = torch.where(z > 0, grad.double(), torch.zeros_like(z))
    fx, fw = gm * t.double(), (gm * s.double()[:, None]).t()
    rx, rw = fx @ p, fw @ q
    assert ((gx.cpu().double() - rx).abs() <= float_bound(fx, p, rx, dtype)).all()
    assert ((gw.cpu().double() - rw).abs() <= float_bound(fw, q, rw, F32)).all()
    assert ((gb.cpu().double() - gm.sum(0)).abs() <= (m + 1) * 2.0 ** -24 * gm.abs().sum(0) + 1e-45).all()
    # the same from the single calls
    c, a = ops.quantize_rows_i8(leaves[0])
    wc, b = ops.quantize_rows_i8(leaves[1])
    z = ops.matmul_i8(c, a, wc, b, leaves[2], True, dtype)
    same_bits(z, y)
    for u, v in zip(ops.linear_i8_backward(grad.to(dev), z, c, a, wc, b, dtype, F32), (gx, gw, gb)):
        same_bits(u, v)


# ------------------------------------------------------------------------------------------ modules as a user wires them
def _heads(dev, int8, rep=24, classes=3):
    from objectdetection_amd.ROIHead import FasterRCNNPredictor, TwoMLPHead
    torch.manual_seed(5)
    return TwoMLPHead(3 * 49, rep, int8=int8).to(dev), FasterRCNNPredictor(rep, classes, int8=int8).to(dev)


@gpu
def test_hooks_run_as_on_the_float_modules(dev):
    """Forward hooks and pre-hooks of the layers inside see what Linear's see (the sums, not what the ReLU leaves), may change
    it, and leave results as they are without them; gradients too, to the bit but for what the predictor's two layers sum in
    one product or in two."""
    head, pred = _heads(dev, True)
    x = features(20, 3 * 49, 3).reshape(20, 3, 7, 7).to(dev).requires_grad_()
    leaves = [x] + list(head.parameters()) + list(pred.parameters())

    def run():
        cls, reg = pred(head(x))
        # the head's gradients from its own output: the predictor's sums would differ in their last bits
        y = head(x)
        return [cls, reg] + list(torch.autograd.grad(y.square().sum(), leaves[:5])) + list(
            torch.autograd.grad(cls.square().sum() + reg.sum(), leaves[5:]))
    plain = run()
    seen, handles = {}, []
    for name, layer in (("fc1", head.fc1), ("fc2", head.fc2), ("cls", pred.cls_score), ("reg", pred.bbox_pred)):
        handles.append(layer.register_forward_hook(lambda m, i, o, name=name: seen.setdefault(name, (m, i[0], o)) and None))
        handles.append(layer.register_forward_pre_hook(lambda m, i, name=name: seen.setdefault("pre " + name, i) and None))
    for u, v in zip(run(), plain):
        same_bits(u, v)
    assert set(seen) == {"fc1", "fc2", "cls", "reg", "pre fc1", "pre fc2", "pre cls", "pre reg"}
    for name, layer in (("fc1", head.fc1), ("fc2", head.fc2), ("cls", pred.cls_score), ("reg", pred.bbox_pred)):
        module, inp, out = seen[name]
        assert module is layer and inp is seen["pre " + name][0]
        q, s = plain_codes(inp)
        p, t = plain_codes(layer.weight)
        same_bits(out, plain_product(q, s, p, t, layer.bias.detach().cpu(), False, F32))
    assert (seen["fc1"][2] < 0).any()
    mid = head(x).detach().requires_grad_()
    up = torch.randn((20, 15), generator=torch.Generator().manual_seed(1))
    hooked, = torch.autograd.grad(torch.cat(pred(mid), 1), mid, up.to(dev))
    for h in handles:
        h.remove()
    fused, = torch.autograd.grad(torch.cat(pred(mid), 1), mid, up.to(dev))
    p, t = plain_codes(torch.cat([pred.cls_score.weight, pred.bbox_pred.weight]))
    f = up.double() * t.double()
    ref = f @ p
    bound = float_bound(f, p, ref, F32)
    assert ((fused.cpu().double() - ref).abs() <= bound).all()
    # two sums, each within the bound of its part, rounded to fp32 and added
    parts = [(f[:, :3], p[:3]), (f[:, 3:], p[3:])]
    bound = sum(float_bound(u, v, u @ v, F32) for u, v in parts) + 2.0 ** -24 * ref.abs() * (1 + 2.0 ** -20) + bound * 2.0 ** -24
    assert ((hooked.cpu().double() - ref).abs() <= bound).all()
    h = head.fc1.register_forward_pre_hook(lambda m, i: (i[0] * 2,))
    same_bits(head(x), head.fc2(head.fc1(x.flatten(1)).relu()).relu())
    doubled = head(x)
    h.remove()
    assert not torch.equal(head(x), doubled)
    calls = []
    h = head.fc2.register_full_backward_hook(lambda m, gi, go: calls.append(go[0].shape) and None)
    torch.autograd.grad(head(x).sum(), x)
    assert calls == [(20, 24)]
    h.remove()


@gpu
@pytest.mark.filterwarnings("ignore")
def test_weight_norm_and_replaced_layers(dev):
    """A weight that a pre-hook or a parametrisation computes is computed on every call, and a layer put in another's place is
    the one that runs."""
    head, pred = _heads(dev, True)
    x = features(9, 3 * 49, 4).to(dev)
    before = head(x)
    torch.nn.utils.weight_norm(head.fc1)
    torch.nn.utils.parametrizations.weight_norm(pred.bbox_pred)
    with torch.no_grad():
        head.fc1.weight_g.mul_(2)
        pred.bbox_pred.parametrizations.weight.original0.mul_(2)
    y = head(x)
    assert not torch.equal(y, before)
    q, s = plain_codes(x)
    first = head.fc1(x)
    p, t = plain_codes(head.fc1.weight)  # as its pre-hook has just left it
    same_bits(first, plain_product(q, s, p, t, head.fc1.bias.detach().cpu(), False, F32))
    assert torch.equal(head.fc1.weight, torch._weight_norm(head.fc1.weight_v, head.fc1.weight_g, 0))
    cls, reg = pred(y)
    wanted = [head.fc1.weight_g, head.fc1.weight_v, pred.bbox_pred.parametrizations.weight.original0, pred.cls_score.weight]
    for g in torch.autograd.grad(reg.square().sum() + cls.square().sum(), wanted):
        assert torch.isfinite(g).all() and g.any()
    head.fc2 = torch.nn.Sequential(head.fc2, torch.nn.Tanh())
    assert (head(x) < 1).all()


def test_layers_follow_a_choice_made_late():
    """int8 set on a module that was built, or pickled, before the choice: its own Linear layers follow, here and back."""
    import copy
    import pickle
    from objectdetection_amd import _lib
    from objectdetection_amd.ROIHead import FasterRCNNPredictor, TwoMLPHead
    x = torch.ones((2, 8))
    for make in (lambda i: TwoMLPHead(8, 4, int8=i), lambda i: FasterRCNNPredictor(8, 3, int8=i)):
        torch.manual_seed(0)
        module = make(False)
        first = module(x)
        for other in (module, copy.deepcopy(module), pickle.loads(pickle.dumps(module))):
            other.int8 = True
            with pytest.raises(_lib.FrcnnError):  # the 8-bit layers have no CPU form
                other(x)
            assert all(type(layer) is torch.nn.Linear for layer in other.children())  # they may be another module's too
            for layer in list(other.children()):
                layer.register_forward_hook(lambda m, i, o: None)
            with pytest.raises(_lib.FrcnnError):
                other(x)
            other.int8 = False
            for u, v in zip(other(x), first):
                assert torch.equal(u, v)
        built = make(True)
        assert all(isinstance(layer, torch.nn.Linear) for layer in built.children())
        with pytest.raises(_lib.FrcnnError):
            built(x)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, torch.float64])
def test_served_head_passes_the_gradient_of_its_input(dev, dtype):
    """In eval mode, as the float head does there: what the head in training form gives for the same weights, to the bit.
    Rows behind a device-side count get none."""
    from objectdetection_amd.ROIHead import Int8FasterRCNNPredictor, Int8Linear, Int8TwoMLPHead
    head, pred = _heads(dev, True)
    served, served_pred = Int8TwoMLPHead.from_float(head).eval(), Int8FasterRCNNPredictor.from_float(pred).eval()
    x = features(50, 3 * 49, 6, dtype, dev).requires_grad_()
    up = torch.randn((50, 15), generator=torch.Generator().manual_seed(2)).to(dev)

    def gradient(h, p, *rows):
        y = torch.cat(p(h(x if h is served else x.to(F32) if dtype == torch.float64 else x, *rows), *rows), 1)
        return y, torch.autograd.grad(y, x, up.to(y.dtype))[0]
    (y, got), (ref_y, ref) = gradient(served, served_pred), gradient(head, pred)
    assert got.dtype == dtype and got.any()
    same_bits(y, ref_y)
    same_bits(got, ref)
    with torch.no_grad():
        x[31:] = float("nan")
    y, part = gradient(served, served_pred, torch.tensor([31], device=dev))
    same_bits(y[:31], ref_y[:31])
    same_bits(part[:31], ref[:31])
    assert (part[31:] == 0).all()
    layer = Int8Linear.from_float(head.fc2.weight).eval()
    z = torch.ones((4, 24), device=dev, requires_grad=True)
    gz, = torch.autograd.grad(layer(z, out_dtype=F16).sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        gz.sum().backward()
    out = layer(z)
    layer.codes.zero_()  # weights loaded between the two halves
    with pytest.raises(RuntimeError):
        out.sum().backward()
    with pytest.raises(RuntimeError):
        layer.train()(z)
    layer = Int8Linear.from_float(head.fc2.weight, relu=True).eval()
    many = torch.randn((140001, 24), generator=torch.Generator().manual_seed(3)).to(dev).requires_grad_()  # more than a call takes
    out = layer(many)
    up = torch.randn((140001, 24), generator=torch.Generator().manual_seed(4)).to(dev)
    rows, = torch.autograd.grad(out, many, up)
    for lo, hi in ((0, 500), (131000, 131500), (139900, 140001)):
        part = many[lo:hi].detach().requires_grad_()
        same_bits(rows[lo:hi], torch.autograd.grad(layer(part), part, up[lo:hi])[0])
    gz, = torch.autograd.grad(layer(z[:0]).sum(), z)
    assert not gz.any()


def test_backward_entry_takes_no_codes_of_x_for_its_gradient_alone():
    """dL/dx needs the weights' codes only; the other two refuse to go without those of x."""
    from objectdetection_amd import _lib
    lib = _lib.load()
    p, null = ctypes.c_void_p(4096), ctypes.c_void_p(0)  # never dereferenced: refused on the host

    def bw(gx, gw, gb, ws=p):
        return lib.frcnn_linear_i8_backward(p, 0, 4, null, 0, null, 32, null, p, 32, p, 4, 4, 32, gx, 0, gw, 0, gb, ws, 16, null)
    for wanted in ((p, p, null), (p, null, p), (null, p, null), (null, null, p)):
        assert bw(*wanted) == -1 and b"null" in lib.frcnn_last_error_string()
    assert bw(p, null, null) == -2 and b"workspace" in lib.frcnn_last_error_string()


@gpu
@pytest.mark.parametrize("count,rows", [((1 << 32) + 3, 20), (-(1 << 32) + 5, 0), (1 << 62, 20), (7, 7), (-1, 0), (2.0 ** 40, 20)])
def test_counts_past_32_bits(dev, count, rows):
    """A row count of 64 bits is clamped to the rows that there are, like one of 32."""
    from objectdetection_amd import ops
    x = features(20, 70, 8).to(dev)
    wc, ws = ops.quantize_rows_i8(torch.randn((6, 70), generator=torch.Generator().manual_seed(1)).to(dev))
    assert int(ops._i8_count(torch.tensor([count], device=dev), "count", dev).clamp(max=20)) == rows
    out = ops.linear_i8(x, wc, ws, n_rows=torch.tensor([count], device=dev))
    same_bits(out[:rows], ops.linear_i8(x, wc, ws)[:rows])


# ------------------------------------------------------------------------- training and quantising rows of every length
@gpu
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (F32, F16), (F16, F16)])
@pytest.mark.parametrize("m,n,k", [(300, 130, 12545), (520, 260, 25088), (40, 70, 33001), (20, 70, 70001), (1100, 40, 2049)])
def test_training_of_long_rows(dev, m, n, k, dtype, wdtype, relu):
    """Sums of the forward call split over workgroups and joined, both operands quantised by the forms for long rows (in one
    launch, in two where their types differ, by two passes), gradients over many tiles of k."""
    _against_the_formulas(dev, m, n, k, dtype, wdtype, relu)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k", [65537, 70003, 131072])
def test_quantize_rows_in_two_passes(dev, k, dtype):
    """Rows too long for the registers in every type: the ends of the type, a row of zeros, Inf and NaN in the last element, an
    odd offset, codes on an odd stride, a row behind the count."""
    from objectdetection_amd import _lib, ops
    fin = torch.finfo(dtype)
    base = features(8, k + 3, k, torch.float64)
    base[:, k] = 1.0
    for i, top in enumerate((fin.max, fin.tiny, fin.tiny * fin.eps * 5, 0.0)):
        base[i] *= top / base[i].abs().max()
    base = base.to(dtype)
    base[4, k], base[5, k] = float("inf"), float("nan")
    base[6, 2::3] *= -1
    ref, ref_scale = plain_codes(base[:, 1:k + 1])
    on = base.to(dev)[:, 1:k + 1]
    codes, scale = ops.quantize_rows_i8(on)
    assert torch.equal(codes.cpu().double(), ref)
    same_bits(scale, ref_scale)
    odd = torch.full((8, k + 2 - k % 2 + 1), 77, dtype=torch.int8, device=dev)
    scale = torch.full((8,), 5.0, device=dev)
    P = ctypes.c_void_p
    n = torch.tensor([7], dtype=torch.int32, device=dev)
    assert _lib.load().frcnn_quantize_rows_i8(P(on.data_ptr()), ops._I8_TYPES[dtype], on.stride(0), 8, k, P(n.data_ptr()),
                                              P(odd.data_ptr()), odd.stride(0), P(scale.data_ptr()),
                                              P(torch.cuda.current_stream().cuda_stream)) == 0
    assert torch.equal(odd.cpu()[:7, :k].double(), ref[:7]) and (odd[:, k:] == 77).all() and (odd[7] == 77).all()
    same_bits(scale[:7], ref_scale[:7])
    assert scale[7] == 5


# --------------------------------------------------------------------------------------------------- captured and side by side
@gpu
@pytest.mark.parametrize("m,n,k", [(300, 130, 12545), (257, 1030, 12545)])
def test_captured_training_of_long_rows(dev, m, n, k):
    """Forward and backward with split sums and by large tiles, and the served layer's gradient behind a row count, in one
    graph; replayed on new inputs with eager work between, each against the eager result; another graph's workspaces beside
    it."""
    from objectdetection_amd import ops
    g = torch.Generator().manual_seed(m)
    x = features(m, k, 41).to(dev).requires_grad_()
    w = (0.05 * torch.randn((n, k), generator=g)).to(dev).requires_grad_()
    b = torch.randn((n,), generator=g).to(dev).requires_grad_()
    up = torch.randn((m, n), generator=g).to(dev)
    wc, ws = ops.quantize_rows_i8(w)
    count = torch.tensor([m - 7], dtype=torch.int32, device=dev)

    def train():
        y = ops.LinearI8.apply(x, w, b, True)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), up)

    def serve():
        y = ops.FrozenLinearI8.apply(x, wc, ws, b.detach(), True, None, count)
        # rows of the output behind the smallest count, m - 51, are unspecified; those of the gradient are zeros
        return y.detach()[:m - 51], torch.autograd.grad(y, x, up)[0]
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), serve()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for step in (train, serve):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held, step))
    for i in range(4):
        with torch.no_grad():
            x.copy_(features(m, k, 50 + i).to(dev))
            w.mul_(-0.5)
            up.neg_()
            count.sub_(11)
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, held, step in graphs:
            got = [t.clone() for t in held]
            for u, v in zip(got, step()):
                same_bits(u, v)


@gpu
def test_training_on_two_streams(dev):
    """Two training steps at once on streams of their own, with inputs of their own."""
    from objectdetection_amd import ops
    steps, eager, got = [], [], [[], []]
    for i in range(2):
        leaves = [features(300, 12545, 60 + i).to(dev).requires_grad_(),
                  torch.randn((130, 12545), generator=torch.Generator().manual_seed(i)).to(dev).requires_grad_()]
        steps.append(lambda leaves=leaves: torch.autograd.grad(ops.LinearI8.apply(*leaves, None, True).square().sum(), leaves))
        eager.append(steps[i]())
    streams = [torch.cuda.Stream(device=dev) for _ in steps]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(steps[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for grads in got[i]:
            for u, v in zip(grads, eager[i]):
                same_bits(u, v)
