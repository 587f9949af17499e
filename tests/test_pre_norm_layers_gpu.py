"""The kernels of pre-norm layers against their formulas in 64 bits: residual + RMS norm (storage type and 8 bits), Dense on
4-bit weights, attention with a sliding window and sinks, and a run of them as a model makes it.

Tolerances count roundings.  u = 2^-24 is half a step of fp32 relative to the value, 2^-11 of fp16; a sum of n terms that
are added in fp32 in any order is off by at most (n - 1) u times the sum of their magnitudes."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}
SMALL = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25}   # half a step among the subnormals
TYPES = {"f32": torch.float32, "f16": torch.float16}


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the -m gpu tests must run on the MI355X box")
    from cubert_amd import kernels
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def within(got, want, bound, what):
    """|got - want| <= bound element by element (want and bound in 64 bits)."""
    torch.cuda.synchronize()
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), "%s: off by %.3g where %.3g is allowed, %d of %d elements" % (
        what, float(off.nan_to_num(math.inf).max()), float(bound.flatten()[off.nan_to_num(math.inf).argmax()]),
        int((~(off <= bound)).sum()), off.numel())


# ---------------------------------------------------------------------------- residual + RMS norm

NORM_SIZES = [(1, 1), (1, 768), (3, 1024), (2, 63), (5, 100), (7, 777), (4, 1000), (9, 2048), (2, 4096), (3, 4100), (2, 8192), (1, 12345),
              (2, 32768), (300, 256), (1029, 1028), (65, 129)]


def norm_reference(x, residual, gamma, eps):
    s = x.double() + (residual.double() if residual is not None else 0)
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, rstd, gamma.double() * s * rstd


def norm_bound(y, hidden, t):
    # s: 1 rounding; the sum of squares of values off by u each: hidden + 2, of which the root takes half; mean, eps, root, reciprocal:
    # 5 at most (reciprocal and root may be two steps off); two products
    return y.abs() * ((hidden + 2) / 2 + 9) * U + y.abs() * (HALF[t] if t != torch.float32 else 0) + 2 * SMALL[t]


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("rows,hidden", NORM_SIZES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_rms_norm(K, t, rows, hidden, with_residual):
    t, g = TYPES[t], gen(rows * 7 + hidden)
    x, gamma = (3 * normal(g, rows, hidden)).to(t), (1 + 0.2 * normal(g, hidden)).to(t)
    residual = normal(g, rows, hidden).to(t) if with_residual else None
    out, total = K.res_rms_norm(x, residual, gamma, 1e-5)
    s, _, y = norm_reference(x, residual, gamma, 1e-5)
    within(out, y, norm_bound(y, hidden, t), "out")
    if with_residual:
        # exact: one rounding of the fp32 sum, and of that to the storage type
        assert torch.equal(total, (x.float() + residual.float()).to(t))
    else:
        assert total is None


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("rows,hidden", NORM_SIZES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_rms_norm_8_bits(K, t, rows, hidden, with_residual):
    t, g = TYPES[t], gen(rows * 5 + hidden)
    x, gamma = (3 * normal(g, rows, hidden)).to(t), (1 + 0.2 * normal(g, hidden)).to(t)
    residual = normal(g, rows, hidden).to(t) if with_residual else None
    codes, scales, total = K.res_rms_norm_i8(x, residual, gamma, 1e-5)
    # the codes are a matter of fp32 operations on single elements: equal, to the last one
    s = x.float().cpu().numpy()
    s = s + residual.float().cpu().numpy() if with_residual else s
    p = gamma.float().cpu().numpy() * s
    top = np.abs(p).max(1, keepdims=True)
    assert np.array_equal(codes.cpu().numpy(), np.rint(p * (np.float32(127) / top)).astype(np.int8))
    if with_residual:
        assert torch.equal(total, (x.float() + residual.float()).to(t))
    _, rstd, y = norm_reference(x, residual, gamma, 1e-5)
    want = y.abs().amax(1) / 127
    within(scales, want, want * ((hidden + 2) / 2 + 11) * U, "scales")
    # what the codes stand for is the norm within half a code, and fp32's roundings of up to 127 of them
    within(codes.double() * want[:, None], y, want[:, None] * (0.5 + 127 * 8 * U) + y.abs() * 8 * U, "values")


# so many rows that a wavefront has one to itself, of one, two and four runs of its lanes, and of more, or of no whole pieces
MANY_ROWS = [(2300, 256), (2048, 512), (2051, 1000), (2049, 1024), (2100, 1792), (2050, 2048), (2049, 4104), (2050, 1001)]


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("rows,hidden", MANY_ROWS)
@pytest.mark.parametrize("with_residual", [False, True])
def test_rms_norm_of_many_rows(K, t, rows, hidden, with_residual):
    test_rms_norm(K, t, rows, hidden, with_residual)
    test_rms_norm_8_bits(K, t, rows, hidden, with_residual)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("hidden", [64, 100, 1024, 5000])
def test_rms_norm_of_rows_without_a_norm(K, t, hidden):
    t = TYPES[t]
    x = torch.ones(6, hidden, device="cuda", dtype=t)
    x[0] = 0
    x[1, hidden // 2] = math.nan
    x[2, 0] = math.inf
    x[3, hidden - 1] = -math.inf
    x[4] = 2.0 ** -24 if t == torch.float16 else 2.0 ** -140     # the smallest values there are
    gamma = torch.ones(hidden, device="cuda", dtype=t)
    codes, scales, _ = K.res_rms_norm_i8(x, None, gamma, 1e-6)
    out, _ = K.res_rms_norm(x, None, gamma, 1e-6)
    codes, scales, out = codes.cpu(), scales.cpu(), out.cpu()
    assert (codes[0] == 0).all() and scales[0] == 0 and (out[0] == 0).all()
    for row in (1, 2, 3):
        assert (codes[row] == 0).all() and math.isnan(scales[row])
        assert math.isnan(out[row][~torch.isfinite(x[row].cpu())][0])
    assert (codes[4:] == 127).all()
    assert abs(float(scales[5]) * 127 - 1) < 1e-5
    assert (out[5].float() - 1).abs().max() < 1e-3
    # a row of zeros has no direction: its norm is zero, whatever is added below the root
    codes, scales, _ = K.res_rms_norm_i8(x, None, gamma, 0.0)
    out, _ = K.res_rms_norm(x, None, gamma, 0.0)
    assert bool((codes[0] == 0).all()) and float(scales[0]) == 0 and bool((out[0] == 0).all())
    assert bool(torch.isnan(out[1]).all()) and math.isnan(scales[1])


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("rows,hidden", [(3, 64), (3, 100), (3, 1024), (3, 5000), (2050, 1024), (2, 8192)])
def test_rms_norm_by_a_gamma_that_is_not_finite(K, t, rows, hidden):
    """Rows that such a gamma leaves no norm have scale NaN and codes 0, wherever in the row it stands; rows that are 0 there too."""
    t, g = TYPES[t], gen(hidden)
    x = normal(g, rows, hidden).to(t)
    for at in (0, hidden // 3, hidden - 1):
        for bad in (math.nan, math.inf, -math.inf) + ((2.0 ** 127,) if t == torch.float32 else ()):
            gamma = torch.ones(hidden, device="cuda", dtype=t)
            gamma[at] = bad
            y = x.clone()
            y[:, at] = 8                                   # (8 * 2^127 is beyond fp32, and its square is not)
            y[1, at] = 0
            codes, scales, _ = K.res_rms_norm_i8(y, None, gamma)
            none = torch.ones(rows, dtype=torch.bool, device="cuda")
            none[1] = bad != 2.0 ** 127                    # (0 times it is 0)
            assert bool((codes[none] == 0).all()) and bool(torch.isnan(scales[none]).all()), (at, bad)
            assert bool(torch.isfinite(scales[~none]).all())


def test_rms_norm_in_place(K):
    """The sum may be written over either input, as the C interface says."""
    from cubert_amd._lib import lib
    g = gen(1)
    for hidden in (100, 768, 4096, 20000):
        x, r = normal(g, 5, hidden), normal(g, 5, hidden)
        gamma = 1 + 0.1 * normal(g, hidden)
        want, total = K.res_rms_norm(x, r, gamma)
        codes, scales, _ = K.res_rms_norm_i8(x, r, gamma)
        stream = torch.cuda.current_stream().cuda_stream
        for over in (0, 1):
            a, b, out = x.clone(), r.clone(), torch.empty_like(x)
            rc = lib().cubert_res_rms_norm_f32(a.data_ptr(), b.data_ptr(), gamma.data_ptr(), 1e-6, (a, b)[over].data_ptr(),
                                               out.data_ptr(), 5, hidden, stream)
            assert rc == 0 and torch.equal(out, want) and torch.equal((a, b)[over], total)
            a, b, out, s = x.clone(), r.clone(), torch.empty_like(codes), torch.empty_like(scales)
            rc = lib().cubert_res_rms_norm_i8_f32(a.data_ptr(), b.data_ptr(), gamma.data_ptr(), 1e-6, (a, b)[over].data_ptr(),
                                                  out.data_ptr(), s.data_ptr(), 5, hidden, stream)
            assert rc == 0 and torch.equal(out, codes) and torch.equal(s, scales) and torch.equal((a, b)[over], total)


def test_rms_norm_at_any_address(K):
    """Rows that start anywhere an element may."""
    g = gen(2)
    for t in (torch.float32, torch.float16):
        for hidden in (768, 1000, 33):
            for shift in (1, 2, 3, 5):
                held = normal(g, 2 * 3 * hidden + 8 + hidden).to(t)
                x, r = held[shift:shift + 3 * hidden].view(3, hidden), held[3 * hidden + 1:6 * hidden + 1].view(3, hidden)
                gamma = held[6 * hidden + shift:7 * hidden + shift]
                out, total = K.res_rms_norm(x, r, gamma)
                want, t2 = K.res_rms_norm(x.clone(), r.clone(), gamma.clone())
                codes, scales, _ = K.res_rms_norm_i8(x, r, gamma)
                codes2, scales2, _ = K.res_rms_norm_i8(x.clone(), r.clone(), gamma.clone())
                _, _, y = norm_reference(x, r, gamma, 1e-6)
                within(out, y, norm_bound(y, hidden, t), "out")
                within(want, y, norm_bound(y, hidden, t), "out")
                assert torch.equal(total, t2) and torch.equal(codes, codes2)
                within(scales, scales2.double(), scales2.double() * (hidden + 24) * U, "scales")


# ---------------------------------------------------------------------------- Dense on 4-bit weights

DENSE_SIZES = [  # tokens, width, features, group
    (1, 32, 1, 32), (1, 64, 16, 64), (1, 128, 17, 128), (2, 96, 40, 32), (3, 768, 2304, 64), (1, 1024, 4096, 128), (5, 4096, 100, 32),
    (16, 768, 768, 128), (17, 640, 50, 64), (31, 1024, 33, 32), (32, 256, 260, 128), (33, 768, 129, 64), (48, 512, 64, 128),
    (64, 4096, 768, 128), (65, 160, 47, 32), (100, 1056, 77, 32), (130, 384, 200, 128), (4, 8192, 48, 128), (9, 8160, 24, 32)]


def unpack(codes):
    c = torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1).to(torch.int16)
    return torch.where(c > 7, c - 16, c)


def weights(g, features, width, group):
    codes = torch.randint(0, 256, (features, width // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.002 + 0.01 * torch.rand(features, width // group, generator=g, device="cuda")).half()
    w = unpack(codes).double() * scales.double().repeat_interleave(group, 1)
    return codes, scales, w


def gelu(y):
    return 0.5 * y * torch.erfc(-y / math.sqrt(2))


def dense_bound(x, w, y, width, group, gelu_too, t):
    """x, w in 64 bits.  A group's products are added in fp32 (its terms may be three per element, of an fp32 x in pieces), scaled,
    and the groups added: 3 group + width / group + 6 roundings at most of the sum of magnitudes."""
    off = (x.abs() @ w.abs().t()) * (3 * group + width / group + 6) * U + y.abs() * 4 * U
    if gelu_too:
        # its slope is at most 1.13; the formula's own error is 1e-7 |y| (activations.h), its evaluation 8 roundings
        off = 1.13 * off + y.abs() * (1e-7 + 8 * U)
        y = gelu(y)
    return y, off + (y.abs() + off) * (HALF[t] if t != torch.float32 else U) + SMALL[t]


@pytest.mark.parametrize("tokens,width,features,group", DENSE_SIZES)
@pytest.mark.parametrize("x_type,t", [("f32", "f32"), ("f16", "f16"), ("i8", "f32"), ("i8", "f16")])
@pytest.mark.parametrize("plain", [True, False])
def test_dense_w4(K, tokens, width, features, group, x_type, t, plain):
    g, t = gen(tokens + width + features), TYPES[t]
    codes, scales, w = weights(g, features, width, group)
    packed = K.w4_pack(codes, scales, group)
    bias = None if plain else normal(g, features).to(t)
    if x_type == "i8":
        x = torch.randint(-127, 128, (tokens, width), generator=g, device="cuda", dtype=torch.int8)
        x_scales = 0.001 + 0.02 * torch.rand(tokens, generator=g, device="cuda")
        out = K.dense_w4_i8(x, x_scales, packed, bias, not plain, t)
        x = x.double() * x_scales.double()[:, None]
    else:
        x = normal(g, tokens, width).to(TYPES[x_type])
        out = K.dense_w4(x, packed, bias, not plain)
        x = x.double()
    y = x @ w.t() + (bias.double() if bias is not None else 0)
    want, bound = dense_bound(x, w, y, width, group, not plain, t)
    assert out.dtype == t
    within(out, want, bound, "out")


# Tokens, width, features, group, so that a workgroup has 32 or 64 features, or 16 and sixteen wavefronts: on both sides of where that
# changes (tiles of 16 features times strips of 16 tokens: 128, 256, 512 and 1024; 8 tokens), with tiles left over and ends inside them
WIDE_DENSE = [(3, 2048, 4000, 128), (8, 1280, 4096, 64), (9, 1280, 2048, 32), (7, 160, 4100, 32), (17, 256, 2064, 64), (8, 128, 8208, 128),
              (5, 416, 12000, 32), (9, 128, 8208, 64), (33, 768, 4100, 128), (1, 128, 16385, 64), (16, 256, 16500, 128), (40, 96, 8200, 32),
              (200, 512, 1300, 64), (64, 1152, 5003, 128)]


@pytest.mark.parametrize("tokens,width,features,group", WIDE_DENSE)
@pytest.mark.parametrize("x_type,t", [("f32", "f32"), ("f16", "f16"), ("i8", "f32"), ("i8", "f16")])
@pytest.mark.parametrize("plain", [True, False])
def test_dense_w4_of_many_features(K, tokens, width, features, group, x_type, t, plain):
    test_dense_w4(K, tokens, width, features, group, x_type, t, plain)


def test_dense_w4_of_many_features_stays_in_its_rows(K):
    """What lies between rows of out stays where a workgroup has 32 or 64 features, and the same call gives the same bits."""
    g = gen(6)
    for tokens, features in ((7, 4100), (20, 8195)):
        codes, scales, w = weights(g, features, 160, 32)
        packed = K.w4_pack(codes, scales, 32)
        x = normal(g, tokens, 160).half()
        held = torch.full((tokens, features + 13), 7.0, device="cuda", dtype=torch.float16)
        K.dense_w4(x, packed, out=held[:, :features])
        want, bound = dense_bound(x.double(), w, x.double() @ w.t(), 160, 32, False, torch.float16)
        within(held[:, :features], want, bound, "out")
        assert bool((held[:, features:] == 7).all())
        for _ in range(3):
            assert torch.equal(K.dense_w4(x, packed), held[:, :features])


def test_dense_w4_rows_apart(K):
    """Rows of x and of out that are longer than what they hold; what lies between rows of out stays."""
    g = gen(3)
    for tokens, width, features in ((3, 256, 50), (40, 128, 33)):
        codes, scales, w = weights(g, features, width, 64)
        packed = K.w4_pack(codes, scales, 64)
        for t in (torch.float32, torch.float16):
            x = normal(g, tokens, width + 64).to(t)[:, 32:32 + width]
            held = torch.full((tokens, features + 13), 7.0, device="cuda", dtype=t)
            assert K.dense_w4(x, packed, out=held[:, :features]) is not None
            want, bound = dense_bound(x.double(), w, x.double() @ w.t(), width, 64, False, t)
            within(held[:, :features], want, bound, "out")
            assert bool((held[:, features:] == 7).all())
            assert K.dense_w4(normal(g, tokens, width + 1).to(t)[:, 1:], packed) is None  # rows of no whole 16 bytes
        x = torch.randint(-127, 128, (tokens, width + 64), generator=g, device="cuda", dtype=torch.int8)[:, 48:48 + width]
        ones = torch.ones(tokens, device="cuda")
        held = torch.full((tokens, features + 13), 7.0, device="cuda")
        K.dense_w4_i8(x, ones, packed, dtype=torch.float32, out=held[:, :features])
        want, bound = dense_bound(x.double(), w, x.double() @ w.t(), width, 64, False, torch.float32)
        within(held[:, :features], want, bound, "out")
        assert bool((held[:, features:] == 7).all())


def test_dense_w4_of_wide_values(K):
    """fp32 rows anywhere in fp32's range, and values that are not finite: they stay in their own rows."""
    g = gen(4)
    codes, scales, w = weights(g, 40, 256, 32)
    w = w.clone()
    packed = K.w4_pack(codes, scales, 32)
    x = normal(g, 8, 256)
    for row, factor in ((0, 2.0 ** 100), (1, 2.0 ** -80), (2, 1e5), (3, 1e-6)):
        x[row] *= factor
    x[4, ::2] *= 2.0 ** 60
    y = x.double() @ w.t()
    want, bound = dense_bound(x.double(), w, y, 256, 32, False, torch.float32)
    within(K.dense_w4(x, packed), want, bound, "out")
    x[5, 17], x[6, 200] = math.inf, math.nan
    out, back = K.dense_w4(x, packed), K.dense_w4(x.clone().half(), packed)
    keep = [0, 1, 2, 3, 4, 7]
    within(out[keep], want[keep], bound[keep], "out")
    code = unpack(codes)[:, 17]
    for f in range(40):
        c = int(code[f])
        assert (math.isnan(out[5, f]) if c == 0 else float(out[5, f]) == math.copysign(math.inf, c)), (f, c, float(out[5, f]))
        assert math.isnan(out[6, f]) and math.isnan(back[6, f])
    assert bool(torch.isfinite(back[7]).all())


def test_dense_w4_is_the_same_twice(K):
    g = gen(5)
    codes, scales, _ = weights(g, 700, 2048, 128)
    packed = K.w4_pack(codes, scales, 128)
    x = normal(g, 20, 2048).half()
    first = K.dense_w4(x, packed)
    for _ in range(5):
        assert torch.equal(K.dense_w4(x, packed), first)
    # a token's result does not depend on its neighbours' values
    y = x.clone()
    y[3] = 100
    again = K.dense_w4(y, packed)
    assert torch.equal(again[:3], first[:3]) and torch.equal(again[4:], first[4:])


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_quantize(K, t, group):
    g, t = gen(group), TYPES[t]
    w = (0.02 * normal(g, 50, 5 * group)).to(t)
    w[3, :group] = 0
    w[4, 0] = 0.5
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    codes, scales = K.w4_quantize(w, group, flag)
    f = w.float().cpu().numpy().reshape(50, 5, group)
    s = (np.abs(f).max(2) / np.float32(7)).astype(np.float16)
    assert np.array_equal(scales.cpu().numpy(), s)
    by = s.astype(np.float32)[:, :, None]
    c = np.clip(np.rint(np.divide(f, by, out=np.zeros_like(f), where=by > 0)), -8, 7)
    got = unpack(codes).cpu().numpy().reshape(50, 5, group)
    assert np.array_equal(got, c)
    assert int(flag) == 0
    # half a step; the largest weight may be beyond code 7 by what the scale's own rounding took
    assert (np.abs(got * by - f) <= by * 0.5 + 7 * by * 2.0 ** -11 + 1e-9).all()
    for bad in (math.nan, math.inf, -math.inf) + ((6e5 if t == torch.float32 else math.inf),):
        v, flag = w.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
        v[7, group + 1] = bad
        codes2, scales2 = K.w4_quantize(v, group, flag)
        assert int(flag) == 1
        assert math.isnan(scales2[7, 1])
        scales2[7, 1] = scales[7, 1]
        assert torch.equal(scales2, scales)
        out = K.dense_w4(torch.ones(1, 5 * group, device="cuda"), K.w4_pack(codes2, K.w4_quantize(v, group)[1], group))
        assert math.isnan(out[0, 7]) and bool(torch.isfinite(out[0, 8:]).all())


# ---------------------------------------------------------------------------- attention with a window and sinks

# batch, q_rows, kv_rows, heads, kv_heads, left, right, sinks, first, lengths, mask
ATTENTION = {
    "one key": (1, 1, 1, 1, 1, -1, -1, 0, None, None, "no"),
    "one query": (2, 1, 300, 4, 2, 100, 0, 4, "end", (300, 77), "no"),
    "all": (2, 70, 70, 2, 2, -1, -1, 0, None, None, "no"),
    "causal": (1, 130, 130, 3, 1, -1, 0, 0, None, None, "no"),
    "encoder": (3, 257, 257, 2, 2, 40, 40, 1, None, (257, 100, 1), "no"),
    "masked encoder": (2, 200, 200, 2, 1, 33, 33, 3, None, None, "padding"),
    "window of one": (1, 100, 100, 2, 2, 0, 0, 0, None, None, "no"),
    "piece": (3, 37, 500, 6, 2, 64, 0, 5, "end", (500, 200, 37), "holes"),
    "piece of seven heads to one": (1, 65, 333, 7, 1, 100, 0, 70, "end", (320,), "holes"),
    "few tokens": (4, 5, 1000, 8, 2, 127, 0, 4, "end", (1000, 999, 64, 5), "no"),
    "before the sequence": (2, 20, 64, 2, 2, 10, 0, 1, "end", (64, 7), "no"),
    "no keys": (2, 3, 50, 2, 1, 10, 0, 0, "end", (50, 0), "no"),
    "nothing left": (2, 40, 40, 2, 2, 5, 5, 0, None, None, "nothing"),
    "sinks alone": (1, 40, 900, 2, 1, 3, 0, 40, "end", (900,), "no"),
    "only to the right": (1, 64, 64, 1, 1, 0, 9, 0, None, None, "no"),
    "sinks beyond the window's end": (1, 50, 80, 2, 1, 4, 2, 30, None, (60,), "no"),
    "long": (1, 1, 5000, 4, 1, -1, 0, 0, "end", (4999,), "holes"),
    "long window": (2, 2, 9000, 8, 1, 4095, 0, 4, "end", (9000, 4500), "no"),
    "behind all keys": (2, 4, 100, 2, 1, 20, 5, 2, (98, 200), (100, 100), "no"),
}

# the same kinds of calls with so many rows that 128 of them share their tiles of keys
WIDE = {
    "wide encoder": (3, 257, 257, 70, 70, 40, 40, 1, None, (257, 100, 1), "no"),
    "wide masked encoder": (2, 200, 200, 100, 50, 33, 33, 3, None, None, "padding"),
    "wide piece": (3, 137, 500, 96, 48, 64, 0, 5, "end", (500, 200, 137), "holes"),
    "wide piece of seven heads to one": (8, 65, 333, 56, 8, 100, 0, 70, "end", (320, 65, 333, 100, 200, 300, 66, 67), "holes"),
    "wide causal": (1, 400, 400, 50, 50, -1, 0, 0, None, None, "no"),
    "wide and all": (4, 150, 150, 24, 24, -1, -1, 0, None, (150, 149, 64, 65), "no"),
    "wide and nothing left": (2, 140, 140, 48, 48, 5, 5, 0, None, None, "nothing"),
    "wide before the sequence": (3, 150, 164, 40, 40, 10, 0, 1, "end", (164, 7, 120), "no"),
    "wide window of one": (2, 129, 129, 49, 49, 0, 0, 0, None, None, "no"),
    "wide, 64 sequences": (64, 140, 150, 4, 2, 30, 0, 2, "end", tuple(150 - 2 * i for i in range(64)), "no"),
    "wide, 70 sequences": (70, 40, 60, 4, 4, 11, 3, 2, None, tuple(max(0, 60 - i) for i in range(70)), "no"),
    "wide and masked from the middle on": (2, 300, 1500, 96, 96, 200, 0, 3, "end", (1500, 1200), "middle"),
    "masked from the middle on": (2, 3, 3000, 4, 2, 700, 0, 3, "end", (3000, 1800), "middle"),
    "wide sinks alone": (5, 40, 900, 80, 20, 3, 0, 40, "end", (900, 100, 800, 40, 41), "no"),
}
ATTENTION.update(WIDE)

# so many rows, and a long axis: 64 of them share their tiles, and in fp32 the axis is cut as well
ATTENTION.update({
    "cut piece": (2, 100, 3000, 8, 4, -1, 0, 3, "end", (3000, 1700), "holes"),
    "cut piece with a window": (1, 300, 2500, 14, 2, 1500, 20, 40, "end", (2477,), "no"),
    "cut causal": (1, 1100, 1100, 4, 4, -1, 0, 0, None, None, "no"),
    "cut encoder": (3, 520, 1030, 6, 6, -1, -1, 0, None, (1030, 33, 0), "no"),
    "cut before the sequence": (2, 200, 2000, 8, 2, 700, 500, 2, "end", (2000, 150), "no"),
    "cut and masked from the middle on": (2, 130, 2100, 9, 3, 1100, 0, 3, "end", (2100, 1500), "middle"),
    "cut and nothing left": (2, 140, 1600, 4, 4, 1100, 5, 0, None, None, "nothing"),
})


def attention_inputs(name, t, size, seed=0):
    batch, q_rows, kv_rows, heads, kv_heads, left, right, sinks, first, lengths, masked = ATTENTION[name]
    g = gen(seed + size + len(name))
    q = normal(g, batch, q_rows, heads, size).to(t)
    k, v = (normal(g, batch, kv_rows, kv_heads, size).to(t) for _ in "kv")
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda") if lengths is not None else None
    if first == "end":
        first = lengths - q_rows
    elif first is not None:
        first = torch.tensor(first, dtype=torch.int32, device="cuda")
    mask = None
    if masked == "padding":
        mask = (torch.arange(kv_rows, device="cuda") < torch.arange(kv_rows, 0, -kv_rows // (batch + 1), device="cuda")[:batch, None]).to(torch.int8)
    elif masked == "holes":
        mask = (torch.rand(batch, kv_rows, generator=g, device="cuda") > 0.2).to(torch.int8) * 3
        mask[0, :kv_rows // 3] = 0
    elif masked == "middle":                               # nothing kept in the last windows but the sinks
        mask = (torch.arange(kv_rows, device="cuda") < torch.tensor([[kv_rows // 2], [kv_rows // 3]], device="cuda")).to(torch.int8)
    elif masked == "nothing":
        mask = torch.zeros(batch, kv_rows, dtype=torch.int8, device="cuda")
        mask[1, 20] = -1
    return q, k, v, dict(left=left, right=right, sinks=sinks, first=first, lengths=lengths, mask=mask)


def visible(q, k, left, right, sinks, first, lengths, mask):
    batch, q_rows, kv_rows = q.shape[0], q.shape[1], k.shape[1]
    p = torch.arange(q_rows, device="cuda") + (first[:, None] if first is not None else torch.zeros(batch, 1, device="cuda", dtype=torch.int64))
    n = lengths if lengths is not None else torch.full((batch,), kv_rows, device="cuda")
    p, n, j = p[:, :, None], n[:, None, None], torch.arange(kv_rows, device="cuda")
    seen = (j < n) & (p >= 0) & (p < n)
    if left >= 0:
        seen = seen & ((j >= p - left) | (j < sinks))
    if right >= 0:
        seen = seen & (j <= p + right)
    if mask is not None:
        seen = seen & (mask[:, None, :] != 0)
    return seen[:, None]                                   # [batch, 1, q_rows, kv_rows]


def attention_reference(q, k, v, alpha=None, **at):
    """The formula in 64 bits, and how far a kernel may be off it."""
    t, size = q.dtype, q.shape[3]
    alpha = size ** -0.5 if alpha is None else alpha
    share = q.shape[2] // k.shape[2]
    seen = visible(q, k, **at)
    hold = seen.any(2)[..., None].transpose(1, 2)          # keys that nobody sees may hold anything: [batch, kv_rows, 1, 1]
    hold = hold.reshape(k.shape[0], k.shape[1], 1, 1)
    k, v = torch.where(hold, k, 0), torch.where(hold, v, 0)
    Q, KT = q.double().permute(0, 2, 1, 3), k.double().repeat_interleave(share, 2).permute(0, 2, 3, 1)
    V = v.double().repeat_interleave(share, 2).permute(0, 2, 1, 3)
    z = (Q @ KT) * alpha
    z = torch.where(seen, z, -math.inf)
    top = z.amax(3, keepdim=True)
    e = torch.where(seen, torch.exp(z - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = e.sum(3, keepdim=True)
    some = torch.where(total > 0, total, 1.0)
    out = (e @ V) / some
    # a score is a sum of `size` products (each of an fp32 operand in up to six pieces), scaled; it and the maximum are held as
    # multiples of log 2 to 2^-24 of the largest
    products = (Q.abs() @ KT.abs()) * abs(alpha)
    slip = torch.where(seen, products, 0.0).amax(3, keepdim=True) * (6 * size + 8) * U
    # a probability: its exponential 2^-22, its rounding to the storage type of the product (among subnormals 2^-25, of a sum that
    # is 1 at least); both sums: the number of keys seen
    count = seen.double().sum(3, keepdim=True)
    each = 2 * slip + 2.0 ** -22 + 2 * count * U + (2.0 ** -11 if t == torch.float16 else 6 * U)
    off = each * ((e @ V.abs()) / some)
    if t == torch.float16:
        off = off + count * 2.0 ** -25 * V.abs().amax((2, 3), keepdim=True) / some
    bound = off + (out.abs() + off) * 2 * HALF[t] + SMALL[t]
    back = lambda x: x.permute(0, 2, 1, 3)                 # noqa: E731
    return back(out), back(bound)


@pytest.mark.parametrize("name", list(ATTENTION))
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
def test_attention_window(K, name, t, size):
    q, k, v, at = attention_inputs(name, TYPES[t], size)
    want, bound = attention_reference(q, k, v, **at)
    got = K.attention_window(q, k, v, **at)
    within(got, want, bound, name)
    blind = ~visible(q, k, **at).any(3)[:, 0]
    assert bool((got[blind] == 0).all())


@pytest.mark.parametrize("name", ["one query", "masked encoder", "piece", "few tokens", "long", "encoder", "nothing left", "wide encoder",
                                  "wide and masked from the middle on", "masked from the middle on",
                                  "wide masked encoder", "wide piece", "wide and nothing left", "cut piece", "cut and nothing left",
                                  "cut encoder", "cut piece with a window", "cut and masked from the middle on"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("filler", [math.nan, math.inf])
def test_attention_window_past_what_it_sees(K, name, t, filler):
    """Keys and values that no query sees may hold anything: behind a sequence, before every window, where the mask is 0."""
    q, k, v, at = attention_inputs(name, TYPES[t], 64)
    want, bound = attention_reference(q, k, v, **at)
    unseen = ~visible(q, k, **at).any(2)[:, 0]             # [batch, kv_rows]
    k, v = k.clone(), v.clone()
    k[unseen], v[unseen] = filler, filler
    within(K.attention_window(q, k, v, **at), want, bound, name)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_window_of_packed_and_padded_rows(K, t):
    """Views of one packed projection, of rows that are longer than their heads, and another scale."""
    g, t = gen(9), TYPES[t]
    for size, heads, kv in ((64, 4, 2), (32, 2, 1), (128, 3, 3)):
        packed = normal(g, 2, 90, heads + 2 * kv + 1, size).to(t)
        q, k, v = packed[:, :, 1:heads + 1], packed[:, :, heads + 1:heads + kv + 1], packed[:, :, heads + kv + 1:]
        at = dict(left=20, right=3, sinks=2, first=None, lengths=torch.tensor([90, 41], dtype=torch.int32, device="cuda"), mask=None)
        want, bound = attention_reference(q, k, v, alpha=-0.03, **at)
        within(K.attention_window(q, k, v, alpha=-0.03, **at), want, bound, "packed")


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_window_of_large_scores(K, t):
    """Scores far apart and far from zero: the softmax picks single keys, and nothing leaves the range."""
    g, t = gen(10), TYPES[t]
    q, k, v = 30 * normal(g, 1, 50, 2, 64).to(t), 30 * normal(g, 1, 400, 2, 64).to(t), normal(g, 1, 400, 2, 64).to(t)
    at = dict(left=200, right=0, sinks=4, first=torch.tensor([350], dtype=torch.int32, device="cuda"), lengths=None, mask=None)
    got = K.attention_window(q, k, v, **at)
    assert bool(torch.isfinite(got).all())
    want, bound = attention_reference(q, k, v, **at)
    within(got, want, bound, "large")


@pytest.mark.parametrize("name", ["one query", "few tokens", "long", "long window", "piece", "masked encoder", "wide piece", "wide masked encoder",
                                  "wide causal", "causal", "encoder", "cut piece", "cut causal", "cut before the sequence"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("where", ["q", "k"])
def test_attention_window_of_no_number(K, name, t, where):
    """What is no number in a query or a key makes none of the results that take it, and of no others."""
    q, k, v, at = attention_inputs(name, TYPES[t], 64)
    want, bound = attention_reference(q, k, v, **at)
    seen, share = visible(q, k, **at)[:, 0], q.shape[2] // k.shape[2]      # [batch, q_rows, kv_rows]
    b, i = (int(x) for x in seen.any(2).nonzero()[seen.any(2).sum() // 2])
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    if where == "q":
        q = q.clone()
        q[b, i, 1, 5] = math.nan
        bad[b, i, 1] = True
    else:
        j = int(seen[b, i].nonzero()[0])
        k = k.clone()
        k[b, j, 0, 63] = math.nan
        bad[b, :, :share] = seen[b, :, j, None]
    got = K.attention_window(q, k, v, **at)
    assert bool(torch.isnan(got[bad]).all())
    within(torch.where(bad[..., None], 0, got), torch.where(bad[..., None], 0.0, want), bound, name)


@pytest.mark.parametrize("name", ["one query", "few tokens", "long", "piece", "masked encoder", "wide piece", "wide masked encoder", "wide causal", "causal",
                                  "encoder", "cut piece", "cut causal", "cut before the sequence"])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("alpha", [0.125, -0.125])
def test_attention_window_of_infinite_keys(K, name, t, size, alpha):
    """An infinite key is a score of -infinity for a query of the other sign, as if it were not there, and no number for the others."""
    q, k, v, at = attention_inputs(name, TYPES[t], size)
    q, k = q.clone(), k.clone()
    q[..., 5] = torch.where(q[..., 5] < 0, -0.5, 0.5).to(q.dtype)
    seen, share = visible(q, k, **at)[:, 0], q.shape[2] // k.shape[2]      # [batch, q_rows, kv_rows]
    b, i = (int(x) for x in seen.any(2).nonzero()[seen.any(2).sum() // 2])
    j = int(seen[b, i].nonzero()[0])
    without = dict(at, mask=torch.ones(k.shape[:2], dtype=torch.int8, device="cuda") if at["mask"] is None else at["mask"].clone())
    without["mask"][b, j] = 0
    want, bound = attention_reference(q, k, v, alpha=alpha, **at)
    want_without, bound_without = attention_reference(q, k, v, alpha=alpha, **without)
    meets = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    meets[b, :, :share] = seen[b, :, j, None]
    none = meets & (q[..., 5] * alpha > 0)
    want, bound = torch.where(meets[..., None], want_without, want), torch.where(meets[..., None], bound_without, bound)
    k[b, j, 0, 5] = math.inf
    got = K.attention_window(q, k, v, alpha=alpha, **at)
    assert bool(torch.isnan(got[none]).all())
    within(torch.where(none[..., None], 0, got), torch.where(none[..., None], 0.0, want), bound, name)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("q_rows,heads", [(1, 2), (3, 8), (50, 60)])
@pytest.mark.parametrize("kv_rows", [9001, 8992, 4624])
def test_attention_window_of_long_padding(K, t, q_rows, heads, kv_rows):
    """Masks that keep nothing from some key on, near and far from the end, at any address: the same as shorter sequences."""
    ends = (0, 1, 15, 500, 513, 528, 4090, 4113, 4624)
    g, t = gen(12), TYPES[t]
    q = normal(g, len(ends), q_rows, heads, 32).to(t)
    k, v = (normal(g, len(ends), kv_rows, 2, 32).to(t) for _ in "kv")
    mask = (torch.arange(kv_rows, device="cuda") < torch.tensor(ends, device="cuda")[:, None]).to(torch.int8)
    at = dict(left=-1, right=-1, sinks=0, first=None, lengths=None, mask=mask)
    got = K.attention_window(q, k, v, **at)
    cut = slice(0, max(ends))
    at["mask"] = mask[:, cut].contiguous()
    for i in range(0, heads, heads // 2):                  # (a head of each key head at a time: the reference is large)
        h = slice(i, i + 1)
        kv = slice(2 * i // heads, 2 * i // heads + 1)
        want, bound = attention_reference(q[:, :, h], k[:, cut, kv], v[:, cut, kv], **at)
        within(got[:, :, h], want, bound, "head %d" % i)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_window_without_scores(K, t):
    """A scale of 0: the mean of what is seen."""
    for name in ("few tokens", "one query", "masked encoder", "wide masked encoder", "long"):
        q, k, v, at = attention_inputs(name, TYPES[t], 64)
        want, bound = attention_reference(q, k, v, alpha=0.0, **at)
        within(K.attention_window(q, k, v, alpha=0.0, **at), want, bound, name)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_window_in_two_graphs(K, t):
    """Calls over a cut axis, two captured and one eager, each with its own partial sums, in turns."""
    calls = [attention_inputs("long", TYPES[t], size, seed) for size, seed in ((64, 1), (64, 2), (128, 3))]
    for q, k, v, at in calls:
        K.attention_window(q, k, v, **at)
    torch.cuda.synchronize()
    graphs = []
    for q, k, v, at in calls[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = K.attention_window(q, k, v, **at)
        graphs.append((graph, out))
    for turn in range(4):
        for q, k, v, at in calls:
            q.copy_(normal(gen(70 + turn), *q.shape))
        for graph, _ in graphs:
            graph.replay()
        eager = K.attention_window(*calls[2][:3], **calls[2][3])
        graphs[0][0].replay()
        got = [out.clone() for _, out in graphs] + [eager]
        torch.cuda.synchronize()
        for out, (q, k, v, at) in zip(got, calls):
            assert torch.equal(out, K.attention_window(q, k, v, **at))
            want, bound = attention_reference(q, k, v, **at)
            within(out, want, bound, "turn %d" % turn)


def test_attention_window_cut_and_uncut(K):
    """A call without room for its pieces runs uncut, with the same result within its bound; and twice gives the same bits."""
    from cubert_amd._lib import lib
    for t in (torch.float32, torch.float16):
        for name in ("long", "long window", "one query", "few tokens", "cut piece", "cut before the sequence"):
            q, k, v, at = attention_inputs(name, t, 64)
            want, bound = attention_reference(q, k, v, **at)
            got = K.attention_window(q, k, v, **at)
            assert torch.equal(K.attention_window(q, k, v, **at), got)
            out = torch.empty_like(q)
            batch, q_rows, heads, size = q.shape
            rc = getattr(lib(), "cubert_attention_window_" + ("f32" if t == torch.float32 else "f16"))(
                q.data_ptr(), heads * size, k.data_ptr(), v.data_ptr(), k.shape[2] * size,
                *(None if at[n] is None else at[n].data_ptr() for n in ("first", "lengths", "mask")), out.data_ptr(), heads * size,
                size ** -0.5, batch, heads, k.shape[2], q_rows, k.shape[1], size, at["left"], at["right"], at["sinks"], None, 0,
                torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            within(out, want, bound, name)


def test_attention_window_lengths_beyond_the_cache(K):
    """Lengths and positions come from the device: ones that no cache holds are cut to what there is."""
    q, k, v, at = attention_inputs("few tokens", torch.float16, 64)
    at["lengths"] = torch.tensor([1000, 2000000000, -5, 5], dtype=torch.int32, device="cuda")
    at["first"] = torch.tensor([995, 990, 0, -2147483648], dtype=torch.int32, device="cuda")
    got = K.attention_window(q, k, v, **at)
    at["lengths"] = torch.tensor([1000, 1000, 0, 5], dtype=torch.int32, device="cuda")
    at["first"] = torch.tensor([995, 990, 0, -100], dtype=torch.int32, device="cuda")
    want, bound = attention_reference(q, k, v, **at)
    within(got, want, bound, "clamped")


def test_attention_window_far_into_a_cache(K):
    """Rows of a cache more than 2^31 elements in."""
    rows, kv, size = 1100000, 16, 128                      # 2.25e9 elements, 4.5 GB
    k = torch.zeros(1, rows, kv, size, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(11)
    n = rows - 3
    near = slice(n - 300, n)
    k[:, near], v[:, near] = normal(g, 1, 300, kv, size).half(), normal(g, 1, 300, kv, size).half()
    v[:, :2] = 1
    q = normal(g, 1, 2, 16, size).half()
    first = torch.tensor([n - 2], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = K.attention_window(q, k, v, left=200, right=0, sinks=2, first=first, lengths=lengths)
    cut_k, cut_v = torch.cat((k[:, :2], k[:, near]), 1), torch.cat((v[:, :2], v[:, near]), 1)
    at = dict(left=200, right=0, sinks=2, first=torch.tensor([300], dtype=torch.int32, device="cuda"), lengths=None, mask=None)
    want, bound = attention_reference(q, cut_k, cut_v, **at)
    within(got, want, bound, "far")


def exact_scores(g, t, batch, q_rows, kv_rows, heads, kv_heads, size):
    """Queries and keys of -1, 0 and 1: every order of summation gives the same scores, whole numbers of at most `size`."""
    q = torch.randint(-1, 2, (batch, q_rows, heads, size), generator=g, device="cuda").to(t)
    return q, torch.randint(-1, 2, (batch, kv_rows, kv_heads, size), generator=g, device="cuda").to(t)


# batch, q_rows, kv_rows, heads, kv_heads, left, right, sinks: single tokens, few rows, 64 rows to a workgroup, 128 rows
ROUNDED_ONCE = [(3, 1, 2000, 8, 2, -1, 0, 0), (2, 4, 90, 8, 4, 3, 0, 1), (2, 300, 300, 12, 12, 2, 0, 1), (4, 300, 300, 32, 32, 2, 0, 0),
                (4, 300, 300, 32, 32, 1, 1, 2), (4, 330, 330, 32, 16, -1, 0, 0)]


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("at", ROUNDED_ONCE)
def test_attention_window_rounds_results_once(K, t, size, at):
    """A result is off by its own rounding and by what fp32 loses on the way, however many rows come with it."""
    batch, q_rows, kv_rows, heads, kv_heads, left, right, sinks = at
    t, g = TYPES[t], gen(size + q_rows)
    q, k = exact_scores(g, t, batch, q_rows, kv_rows, heads, kv_heads, size)
    v = normal(g, batch, kv_rows, kv_heads, size).to(t)
    first = torch.full((batch,), kv_rows - q_rows, dtype=torch.int32, device="cuda")
    at = dict(left=left, right=right, sinks=sinks, first=first, lengths=None, mask=None)
    got = K.attention_window(q, k, v, alpha=0.125, **at)
    want, _ = attention_reference(q, k, v, alpha=0.125, **at)
    share, seen = heads // kv_heads, visible(q, k, **at)
    Q, KT = q.double().permute(0, 2, 1, 3), k.double().repeat_interleave(share, 2).permute(0, 2, 3, 1).contiguous()
    V = v.double().abs().repeat_interleave(share, 2).permute(0, 2, 1, 3).contiguous()
    z = torch.where(seen, (Q @ KT) * 0.125, -math.inf)
    e = torch.exp(z - z.amax(3, keepdim=True))
    total, back = e.sum(3, keepdim=True), lambda x: x.permute(0, 2, 1, 3)
    # An exponent is a whole number times alpha log2(e), at most size / 8 * 1.443, less a maximum that is as large: the factor is off by
    # 2 u of it, the maximum by 3 u, the difference by u of twice that, and e's exponential of that by log 2 times it.
    exponent = math.log(2) * size / 8 * 1.443 * 8 * U
    # An exponential: 2^-22; a probability in two terms of 11 bits: 2^-22; sums of it and of the products: 3 n u.  The same for the sum.
    count = float(seen.sum(3).max())
    off = (e @ V) / total * (2 * exponent + 2.0 ** -21 + 2.0 ** -22 + 4 * count * U)
    if t == torch.float16:  # terms among fp16's subnormals: 2^-25 of the largest probability, for every key
        off = off + 2.0 ** -25 * (seen.double().expand(e.shape) @ V) / total
    off = back(off)
    within(got, want, (want.abs() + off) * HALF[t] + off + SMALL[t], "rounded once")


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("q_rows", [1, 3, 768, 5120])
@pytest.mark.parametrize("at", [0, 70000, 131071])
def test_attention_window_of_a_long_axis_next_to_one_key(K, t, q_rows, at):
    """One key stands so far out that each of 131071 others is less than half of fp16's smallest number next to it; together they
    are 3 thousandths of the result."""
    t, keys, size, score = TYPES[t], 131072, 64, 17.5
    q = torch.ones(1, q_rows, 8, size, device="cuda", dtype=t)
    k, v = torch.zeros(1, keys, 1, size, device="cuda", dtype=t), torch.ones(1, keys, 1, size, device="cuda", dtype=t)
    k[:, at], v[:, at] = 1, 0
    got = K.attention_window(q, k, v, alpha=score / size)
    others = (keys - 1) * math.exp(-score)
    want = torch.full(got.shape, others / (1 + others), dtype=torch.float64, device="cuda")
    # The exponents are score log2(e), in fp32: 6 u of 26; exponentials 2^-22; a lane adds up to half of the keys one by one, each
    # addition off by u of what is there, in the sum and in the products.
    off = want * (math.log(2) * 26 * 6 * U + 2.0 ** -21 + 2 * (keys / 2 + 64) * U)
    if t == torch.float16:
        off = off + keys * 2.0 ** -35
    within(got, want, want * HALF[t] + off + SMALL[t], "others")


@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("batch,heads", [(1, 1), (3, 2), (4, 8)])
def test_attention_window_of_scores_that_cancel(K, size, batch, heads):
    """fp32 scores that are a millionth of the two products that make them: what a product leaves out stays below its own rounding."""
    g, rows = gen(size), 1300
    # numbers just below a step of 8 bits, whose parts below are as large as they get, and any numbers
    step = 1 + torch.randint(1, 9, (2, batch, rows, heads), generator=g, device="cuda") * 2.0 ** -7 - 2.0 ** -23
    some = 1 + torch.rand(2, batch, rows, heads, generator=g, device="cuda") / 16
    x, y = torch.where(torch.arange(rows, device="cuda")[:, None] % 2 == 0, step, some)
    y = y * 2.0 ** 20
    q, k = (torch.zeros(batch, rows, heads, size, device="cuda") for _ in "qk")
    q[..., 0], q[..., 1] = x, 1
    k[..., 0], k[..., 1] = y, -(x * y)
    v = torch.ones_like(k)
    k[:, 0], v[:, 0] = 0, 0                                # the first key has score 0 and value 0; a query sees it and its own
    got = K.attention_window(q, k, v, left=0, right=0, sinks=1, alpha=1.0)
    product = x.double() * y.double()
    want = torch.sigmoid(product - (x * y).double())
    want[:, 0] = 0
    # The product leaves out u of it.  It and the other, as large, meet in the last matrix instruction, whose two sums are off by a step
    # (2 u) each; the instructions before have 2^-7 of that.  A sigmoid's slope is a quarter; exponentials and the quotient: 2^-20.
    bound = 0.25 * 5.25 * U * product + 2.0 ** -20
    within(got[..., 0], want, bound, "cancelled")
    assert bool((got == got[..., :1]).all())


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("rows,heads", [(1, 1), (40, 2), (300, 8), (400, 40)])
@pytest.mark.parametrize("alpha", [0.5, -0.5])
def test_attention_window_of_the_largest_numbers(K, t, rows, heads, alpha):
    """The largest numbers as keys and as values (the nearest in 16 bits to fp32's is infinite), and scores as large as they make."""
    t = TYPES[t]
    most = torch.finfo(t).max
    q, k, v = (torch.zeros(2, rows, heads, 64, device="cuda", dtype=t) for _ in "qkv")
    if t == torch.float32:
        q[..., 0] = 0.25
    else:
        q[:] = most                                        # 64 products of 4.3e9
    up = math.copysign(most, alpha)                        # (a key whose score is above 0)
    k[0], k[1], v[..., :32] = -up, up, 1
    k[:, 0] = 0                                            # a query sees the first key, whose score is 0, its own and the one before
    v[:, 0, :, 32:] = most
    got = K.attention_window(q, k, v, left=1, right=0, sinks=1, alpha=alpha)
    want = torch.zeros(got.shape, dtype=torch.float64, device="cuda")
    want[0, :, :, :32], want[0, :, :, 32:] = 1, most       # scores so low that the first key is all there is, or so high that it is not
    want[1, :, :, :32] = 1
    want[:, 0, :, :32], want[:, 0, :, 32:] = 1, most
    within(got, want, want.abs() * 16 * U, "largest")


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("name", ["one query", "few tokens", "piece", "wide piece", "cut piece", "long"])
@pytest.mark.parametrize("alpha", [2.0 ** 40, -3e38])
def test_attention_window_of_a_large_scale(K, t, name, alpha):
    """Scores that are whole numbers, times so much that only the largest of them count: the mean of their values."""
    q, k, v, at = attention_inputs(name, TYPES[t], 64)
    g = gen(14)
    q, k = exact_scores(g, q.dtype, q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], 64)
    got = K.attention_window(q, k, v, alpha=alpha, **at)
    want, _ = attention_reference(q, k, v, alpha=math.copysign(1e4, alpha), **at)
    # sums of the values that count, in fp32, over as many; one rounding
    count = float(visible(q, k, **at).sum(3).max())
    bound = 4.0 * count * U * float(v.double().abs().max())
    within(got, want, want.abs() * HALF[q.dtype] + bound + SMALL[q.dtype], name)


# ---------------------------------------------------------------------------- streams, graphs, a run of them


def test_on_another_stream_and_replayed(K):
    """A captured step of a layer, replayed with other inputs in place and eager work of the same operators in between."""
    layer = Layer(K, 21, torch.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = normal(gen(1), 3, layer.hidden).half()
        layer.step(x, 40)
    torch.cuda.current_stream().wait_stream(side)
    layer.at(40)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer.step(x, None)
    other = Layer(K, 22, torch.float16)
    for turn in range(4):
        x.copy_(normal(gen(50 + turn), 3, layer.hidden).half())
        layer.at(40 + turn)
        graph.replay()
        got = [o.clone() for o in outs]
        other.step(x, 100)
        torch.cuda.synchronize()
        want = layer.step(x, 40 + turn)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


class Layer(object):
    """One pre-norm layer on 4-bit weights over a cache: 8-bit rows into the packed projection, attention with a window and
    sinks, the output layer, the second norm and the two layers of the intermediate part."""

    hidden, heads, kv, size, wide, window, sinks, room = 256, 4, 2, 64, 512, 30, 3, 128

    def __init__(self, K, seed, t, batch=3):
        g = gen(seed)
        self.K, self.t = K, t
        self.gamma = [(1 + 0.1 * normal(g, self.hidden)).to(t) for _ in range(2)]
        shapes = [((self.heads + 2 * self.kv) * self.size, self.hidden), (self.hidden, self.heads * self.size), (self.wide, self.hidden),
                  (self.hidden, self.wide)]
        self.w, self.packed = [], []
        for features, width in shapes:
            codes, scales = K.w4_quantize(0.05 * normal(g, features, width), 64)
            self.packed.append(K.w4_pack(codes, scales, 64))
            self.w.append(unpack(codes).double() * scales.double().repeat_interleave(64, 1))
        self.bias = (0.1 * normal(g, self.wide)).to(t)
        self.k, self.v = (normal(g, batch, self.room, self.kv, self.size).to(t) for _ in "kv")
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.rows = torch.zeros(batch, dtype=torch.int64, device="cuda")

    def at(self, n):
        """The next token stands at position n of every sequence."""
        self.lengths.fill_(n + 1)
        self.rows.copy_(torch.arange(len(self.rows), device="cuda") * self.room + n)

    def step(self, x, n):
        K, batch = self.K, x.shape[0]
        if n is not None:
            self.at(n)
        codes, scales, _ = K.res_rms_norm_i8(x, None, self.gamma[0])
        qkv = K.dense_w4_i8(codes, scales, self.packed[0], dtype=self.t).view(batch, 1, -1, self.size)
        q, k, v = qkv[:, :, :self.heads], qkv[:, :, self.heads:self.heads + self.kv], qkv[:, :, self.heads + self.kv:]
        self.k.view(-1, self.kv, self.size).index_copy_(0, self.rows, k[:, 0])
        self.v.view(-1, self.kv, self.size).index_copy_(0, self.rows, v[:, 0])
        ctx = K.attention_window(q, self.k, self.v, self.window, 0, self.sinks, first=self.lengths - 1, lengths=self.lengths)
        att = K.dense_w4(ctx.view(batch, -1), self.packed[1])
        y, total = K.res_rms_norm(att, x, self.gamma[1])
        mid = K.dense_w4(y, self.packed[2], self.bias, gelu=True)
        return codes, scales, qkv, ctx, att, y, total, mid, K.dense_w4(mid, self.packed[3])


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_a_layer_step_by_step(K, t):
    """Every stage of a run against 64 bits of what it was given, over single tokens that fill a cache past its window."""
    t = TYPES[t]
    layer = Layer(K, 31, t)
    g = gen(32)
    for n in (0, 1, 2, 33, 34, 35, 127):
        x = normal(g, 3, layer.hidden).to(t)
        codes, scales, qkv, ctx, att, y, total, mid, out = layer.step(x, n)
        _, _, norm = norm_reference(x, None, layer.gamma[0], 1e-6)
        want = norm.abs().amax(1) / 127
        within(codes.double() * want[:, None], norm, want[:, None] * (0.5 + 127 * 8 * U) + norm.abs() * 8 * U, "codes")

        def dense(x, w, out, bias=0.0, gelu_too=False):
            y = x @ w.t() + bias
            ref, bound = dense_bound(x, w, y, w.shape[1], 64, gelu_too, t)
            within(out, ref, bound, "dense")

        dense(codes.double() * scales.double()[:, None], layer.w[0], qkv.view(3, -1))
        at = dict(left=layer.window, right=0, sinks=layer.sinks, first=layer.lengths - 1, lengths=layer.lengths, mask=None)
        ref, bound = attention_reference(qkv[:, :, :layer.heads], layer.k, layer.v, **at)
        within(ctx, ref, bound, "ctx")
        dense(ctx.double().view(3, -1), layer.w[1], att)
        _, _, norm = norm_reference(att, x, layer.gamma[1], 1e-6)
        within(y, norm, norm_bound(norm, layer.hidden, t), "second norm")
        assert torch.equal(total, (att.float() + x.float()).to(t))
        dense(y.double(), layer.w[2], mid, layer.bias.double(), True)
        dense(mid.double(), layer.w[3], out)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_a_prompt_in_pieces_is_the_prompt(K, t):
    """A prompt at once, in pieces and token by token over the same cache give the same rows within the bound of one of them."""
    t = TYPES[t]
    g = gen(41)
    q, k, v = normal(g, 2, 150, 4, 64).to(t), normal(g, 2, 150, 2, 64).to(t), normal(g, 2, 150, 2, 64).to(t)
    at = dict(left=50, right=0, sinks=2, first=None, lengths=None, mask=None)
    want, bound = attention_reference(q, k, v, **at)
    for piece in (150, 64, 7, 1):
        for begin in range(0, 150, piece):
            end = min(begin + piece, 150)
            now = torch.full((2,), begin, dtype=torch.int32, device="cuda")
            got = K.attention_window(q[:, begin:end].contiguous(), k, v, 50, 0, 2, first=now, lengths=now + (end - begin))
            within(got, want[:, begin:end], bound[:, begin:end], "piece %d at %d" % (piece, begin))


def test_wrappers_refuse(K):
    g = gen(51)
    x = normal(g, 4, 64)
    for call in (lambda: K.res_rms_norm(x, x.half(), x[0]), lambda: K.res_rms_norm(x, None, x[0, :32]),
                 lambda: K.res_rms_norm(x.t(), None, x[0]), lambda: K.res_rms_norm(x, x[:2], x[0]),
                 lambda: K.w4_quantize(x, 48), lambda: K.w4_quantize(x, 128)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        K.res_rms_norm(x.double(), None, x[0].double())
    codes, scales = K.w4_quantize(x, 64)
    w = K.w4_pack(codes, scales, 64)
    ints, ones = torch.zeros(2, 64, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda")
    for call in (lambda: K.w4_pack(codes, scales, 32), lambda: K.w4_pack(codes, scales.float(), 64), lambda: K.dense_w4(x[:, :32], w),
                 lambda: K.dense_w4(x, w, bias=x[0, :3]), lambda: K.dense_w4(x, w, bias=x[0, :4].half()), lambda: K.dense_w4_i8(x, ones, w),
                 lambda: K.dense_w4_i8(ints, ones[:1], w), lambda: K.dense_w4(x, w, out=torch.empty(4, 3, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    q, k = normal(g, 2, 3, 4, 64), normal(g, 2, 9, 2, 64)
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: K.attention_window(q, k.half(), k.half()), lambda: K.attention_window(q, k, k[:, :8]),
                 lambda: K.attention_window(q, k[:, :, :1].expand(2, 9, 3, 64), k[:, :, :1].expand(2, 9, 3, 64)),
                 lambda: K.attention_window(q, k, k, lengths=n.long()), lambda: K.attention_window(q, k, k, first=n[:1]),
                 lambda: K.attention_window(q, k, k, mask=torch.zeros(2, 8, dtype=torch.int8, device="cuda")),
                 lambda: K.attention_window(q[:, :, ::2], k, k), lambda: K.attention_window(q, k[:, :7], k[:, :7])):
        with pytest.raises(ValueError):
            call()
    assert K.attention_window(q[..., :48].contiguous(), k[..., :48].contiguous(), k[..., :48].contiguous()) is None
    assert K.attention_window(q[:0], k[:0], k[:0]).shape == (0, 3, 4, 64)
    assert K.dense_w4(x[:0], w).shape == (0, 4)
    assert K.res_rms_norm(x[:0], None, x[0])[0].shape == (0, 64)
    empty = K.attention_window(q, k[:, :0].contiguous(), k[:, :0].contiguous())
    assert bool((empty == 0).all())
