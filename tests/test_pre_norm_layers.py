"""What the kernels of pre-norm layers refuse, and the sizes that callers ask for: no device call is made."""
import pytest

torch = pytest.importorskip("torch")  # before the library: both bring a HIP runtime

BAD_ARGUMENT, UNSUPPORTED = -1, -2
P = 4096  # an aligned address that nothing may read


@pytest.fixture(scope="module")
def L():
    from cubert_amd._lib import lib
    return lib()


def norm(L, t, codes, rows=4, hidden=64, eps=1e-6, x=P, gamma=P, out=P, scales=P):
    if codes:
        return getattr(L, "cubert_res_rms_norm_i8_" + t)(x, P, gamma, eps, P, out, scales, rows, hidden, None)
    return getattr(L, "cubert_res_rms_norm_" + t)(x, P, gamma, eps, P, out, rows, hidden, None)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("codes", [False, True])
def test_rms_norm_refuses(L, t, codes):
    for wrong in (dict(rows=-1), dict(hidden=0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None),
                  dict(gamma=None), dict(out=None)):
        assert norm(L, t, codes, **wrong) == BAD_ARGUMENT, wrong
    if codes:
        assert norm(L, t, codes, scales=None) == BAD_ARGUMENT
    assert norm(L, t, codes, hidden=32769) == UNSUPPORTED
    assert norm(L, t, codes, rows=1 << 26) == UNSUPPORTED                  # more rows than a launch holds
    assert norm(L, t, codes, rows=1 << 24, hidden=1) == UNSUPPORTED
    assert norm(L, t, codes, rows=1 << 22, hidden=32768) == UNSUPPORTED
    assert norm(L, t, codes, rows=0, x=None, out=None) == 0


def dense(L, name, tokens=3, features=40, width=256, x=P, ldx=None, packed=P, group=64, activation=0, out=P, ldo=None, scales=P):
    rows = (x, width if ldx is None else ldx) + ((scales,) if "i8" in name else ())
    return getattr(L, "cubert_dense_w4_" + name)(None, tokens, features, width, *rows, packed, group, None, activation, out,
                                                 features if ldo is None else ldo)


@pytest.mark.parametrize("name", ["f32", "f16", "i8_f32", "i8_f16"])
def test_dense_w4_refuses(L, name):
    for wrong in (dict(tokens=-1), dict(features=0), dict(width=0), dict(x=None), dict(packed=None), dict(out=None), dict(ldx=255),
                  dict(ldo=39), dict(activation=2)) + ((dict(scales=None),) if "i8" in name else ()):
        assert dense(L, name, **wrong) == BAD_ARGUMENT, wrong
    for other in (dict(group=16), dict(group=96), dict(width=96, group=64), dict(x=P + 8), dict(ldx=258), dict(packed=P + 4)):
        assert dense(L, name, **other) == UNSUPPORTED, other
    assert dense(L, name, tokens=0, x=None, out=None) == 0
    assert dense(L, name, tokens=(1 << 31) - 1) == UNSUPPORTED             # more than a launch holds
    assert dense(L, name, tokens=1 << 24, features=(1 << 31) - 1) == UNSUPPORTED


def test_w4_sizes_and_refusals(L):
    # 16 features and 128 columns are 1024 bytes of codes, and 32 bytes of scales for each of their groups
    assert L.cubert_w4_packed_bytes(16, 128, 128) == 1024 + 32
    assert L.cubert_w4_packed_bytes(17, 160, 32) == 4 * (1024 + 4 * 32)
    assert L.cubert_w4_packed_bytes(1, 64, 64) == 1024 + 2 * 32
    assert L.cubert_w4_packed_bytes(32768, 65536, 128) == 2048 * 512 * (1024 + 32)
    for sizes in ((0, 128, 128), (16, 0, 128), (16, 128, 16), (16, 96, 64), ((1 << 31) - 1, 1 << 20, 128)):
        assert L.cubert_w4_packed_bytes(*sizes) == 0
    for t in ("f32", "f16"):
        quantize = getattr(L, "cubert_w4_quantize_" + t)
        assert quantize(None, 16, 128, 64, P, P, None, None) == BAD_ARGUMENT
        assert quantize(P, 16, 128, 64, None, P, None, None) == BAD_ARGUMENT
        assert quantize(P, 0, 128, 64, P, P, None, None) == BAD_ARGUMENT
        assert quantize(P, 16, 100, 64, P, P, None, None) == UNSUPPORTED
    assert L.cubert_w4_pack(P, None, 16, 128, 64, P, None) == BAD_ARGUMENT
    assert L.cubert_w4_pack(P, P, 16, 128, 48, P, None) == UNSUPPORTED
    assert L.cubert_w4_pack(P, P, 16, 128, 64, P + 8, None) == UNSUPPORTED
    assert L.cubert_w4_pack(P, P, (1 << 31) - 1, 1 << 20, 64, P, None) == UNSUPPORTED


def attention(L, t, q=P, ldq=None, k=P, v=P, ldkv=None, ctx=P, ld_ctx=None, batch=2, heads=4, kv_heads=2, q_rows=3, kv_rows=50, size=64,
              left=-1, right=0, sinks=0, alpha=1.0):
    return getattr(L, "cubert_attention_window_" + t)(
        q, heads * size if ldq is None else ldq, k, v, kv_heads * size if ldkv is None else ldkv, None, None, None, ctx,
        heads * size if ld_ctx is None else ld_ctx, alpha, batch, heads, kv_heads, q_rows, kv_rows, size, left, right, sinks, None, 0, None)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_window_refuses(L, t):
    for wrong in (dict(q=None), dict(k=None), dict(v=None), dict(ctx=None), dict(batch=-1), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3),
                  dict(q_rows=-1), dict(kv_rows=-1), dict(size=0), dict(sinks=-1), dict(ldq=255), dict(ldkv=127), dict(ld_ctx=255),
                  dict(kv_rows=1 << 30), dict(q_rows=1 << 30), dict(alpha=float("nan")), dict(alpha=float("inf")), dict(alpha=float("-inf"))):
        assert attention(L, t, **wrong) == BAD_ARGUMENT, wrong
    for other in (dict(size=48), dict(size=256), dict(q=P + 8), dict(k=P + 8), dict(v=P + 8), dict(ctx=P + 8), dict(ldq=258), dict(ldkv=130),
                  dict(ld_ctx=258), dict(ldkv=(1 << 22) + 64), dict(batch=1 << 23), dict(batch=(1 << 31) - 1, kv_heads=4),
                  dict(q_rows=(1 << 30) - 1, heads=4, kv_heads=1), dict(batch=1 << 20, q_rows=1 << 20)):
        assert attention(L, t, **other) == UNSUPPORTED, other
    assert attention(L, t, batch=0, q=None) == 0
    assert attention(L, t, q_rows=0, q=None) == 0


def test_attention_window_partials(L):
    """Floats for the rows of a workgroup, head size + 4 each, per piece of the axis, and none where nothing is cut."""
    for half in (0, 1):
        def floats(batch, heads, kv_heads, q_rows, kv_rows, size, left=-1, right=0, sinks=0):
            return L.cubert_attention_window_partials(half, batch, heads, kv_heads, q_rows, kv_rows, size, left, right, sinks)
        assert floats(1, 16, 2, 1, 131072, 128) == 2 * 128 * 32 * 132
        assert floats(4, 8, 4, 1, 2048, 64) == 16 * 16 * 32 * 68       # 64 tiles of 32 keys, four of them to a piece
        assert floats(4, 8, 4, 1, 8192, 64, left=95) == 0              # 128 keys are one piece
        assert floats(4, 8, 4, 1, 8192, 64, left=96) == 16 * 2 * 32 * 68
        assert floats(1, 4, 4, 1, 128, 64) == 0
        assert floats(512, 12, 12, 1, 4096, 64) == 0
        assert floats(8, 12, 12, 512, 512, 64) == 0
        assert floats(2, 8, 4, 100, 3000, 64) == (32 * 5 * 64 * 68 if not half else 56 * 7 * 32 * 68)
        assert floats(1, 12, 12, 2048, 2048, 64) == (384 * 2 * 64 * 68 if not half else 0)
        assert half or floats(1, 12, 12, 600, 600, 64, right=-1) == 0
        for nothing in ((0, 4, 2, 1, 50, 64), (1, 4, 3, 1, 50, 64), (1, 4, 0, 1, 50, 64), (1, 4, 2, 0, 50, 64), (1, 4, 2, 1, 0, 64),
                        (1, 4, 2, 1, 50, 0), (1 << 30, 1 << 20, 1 << 20, 1, 5000, 64)):
            assert floats(*nothing) == 0


def test_wrappers_refuse_host_tensors():
    from cubert_amd import kernels
    x, g = torch.zeros(2, 64), torch.ones(64)
    with pytest.raises(ValueError):
        kernels.res_rms_norm(x, None, g)
    with pytest.raises(ValueError):
        kernels.w4_quantize(x)
    q = torch.zeros(1, 2, 2, 64)
    with pytest.raises(ValueError):
        kernels.attention_window(q, q, q)


def test_strided_heads_are_recognised():
    from cubert_amd.kernels import _heads_pitch
    packed = torch.zeros(3, 5, 8, 64)
    assert _heads_pitch(packed[:, :, 2:4], "k") == 8 * 64
    assert _heads_pitch(packed[:1, :, :4], "q") == 8 * 64
    assert _heads_pitch(packed[:, :1].contiguous()[:, :, 4:], "q") == 8 * 64
    for wrong in (packed[:, :, ::2], packed[..., ::2], packed.transpose(1, 2), packed[:, 1:4], packed[::2],
                  packed[:, :1].expand(3, 5, 8, 64)):
        with pytest.raises(ValueError):
            _heads_pitch(wrong, "k")


def test_quantize_wants_an_int_to_write_to():
    """4 bytes are written there."""
    from cubert_amd import kernels
    for overflow in (torch.zeros(1, dtype=torch.int8), torch.zeros(1, dtype=torch.bool), torch.zeros(1, dtype=torch.int64),
                     torch.zeros(1), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="int32"):
            kernels.w4_quantize(torch.zeros(2, 64), 64, overflow)


def test_a_negative_number_of_sinks_stays_one(monkeypatch):
    from cubert_amd import kernels
    calls = []
    monkeypatch.setattr(kernels, "_device", lambda *tensors: 0)
    monkeypatch.setattr(kernels, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(kernels, "_run_on", lambda device, name, args: calls.append(args) or True)
    q = torch.zeros(1, 3, 2, 64)
    for sinks, sent in ((4, 4), (0, 0), (-1, -1), (5 - (1 << 32), -1), (1 << 40, 1 << 30)):
        kernels.attention_window(q, q, q, left=7, right=0, sinks=sinks)
        assert calls[-1][-6:-3] == (7, 0, sent), sinks      # left, right, sinks, partials, their number, stream


def test_wrappers_refuse_what_32_bits_do_not_hold():
    """The C interface has 32 bits for sizes and pitches: 2**32 + 64 would arrive as 64."""
    from cubert_amd import kernels

    def empty(*shape, dtype=torch.float16):
        return torch.empty(shape, dtype=dtype, device="meta")

    large = (1 << 32) + 64
    w = kernels.W4Weights(empty(8, dtype=torch.uint8), 16, 64, 64)
    apart = torch.empty_strided((2, 64), (large, 1), dtype=torch.float16, device="meta")
    for call in (lambda: kernels.res_rms_norm(empty(1, large), None, empty(large)),
                 lambda: kernels.res_rms_norm_i8(empty(1, large), None, empty(large)),
                 lambda: kernels.w4_quantize(empty(1, large), 64), lambda: kernels.w4_quantize(empty(large, 64), 64),
                 lambda: kernels.w4_pack(empty(1, large // 2, dtype=torch.uint8), empty(1, large // 64), 64),
                 lambda: kernels.dense_w4(empty(large, 64), w), lambda: kernels.dense_w4(apart, w),
                 lambda: kernels.dense_w4(empty(2, 64), w, out=torch.empty_strided((2, 16), (large, 1), dtype=torch.float16, device="meta")),
                 lambda: kernels.attention_window(empty(1, large, 1, 64), empty(1, 9, 1, 64), empty(1, 9, 1, 64)),
                 lambda: kernels.attention_window(empty(1, 9, 1, 64), empty(1, large, 1, 64), empty(1, large, 1, 64))):
        with pytest.raises(ValueError, match="2\\*\\*31"):
            call()
