"""What the kernels of a key/value cache in pages refuse: no device call is made."""
import pytest

torch = pytest.importorskip("torch")  # before the library: both bring a HIP runtime

BAD_ARGUMENT, UNSUPPORTED = -1, -2
P = 4096  # an aligned address that nothing may read
Q = 8192  # another one
LARGE = (1 << 31) - 1


@pytest.fixture(scope="module")
def L():
    from cubert_amd._lib import lib
    return lib()


def extend(L, table=P, width=8, ld_table=None, lengths=P, counts=P, free=P, free_count=P, places=100, pages=100, page=16, batch=3, rows=2, slots=P, lengths_out=Q,
           free_out=Q):
    return L.cubert_paged_extend(table, width, width if ld_table is None else ld_table, lengths, counts, free, free_count, places, pages, page, batch, rows,
                                 slots, lengths_out, free_out, None)


def cut(L, table=P, width=8, ld_table=None, lengths=P, keep=P, free=P, free_count=P, places=100, pages=100, page=16, batch=3, lengths_out=Q, free_out=Q, work=P):
    return L.cubert_paged_cut(table, width, width if ld_table is None else ld_table, lengths, keep, free, free_count, places, pages, page, batch,
                              lengths_out, free_out, work, None)


@pytest.mark.parametrize("call", [extend, cut])
def test_tables_refuse(L, call):
    for wrong in (dict(table=None), dict(width=0), dict(ld_table=7), dict(lengths=None), dict(free=None), dict(free_count=None), dict(places=0), dict(pages=0), dict(page=0),
                  dict(page=-16), dict(batch=-1), dict(lengths_out=None), dict(free_out=None), dict(lengths_out=P), dict(free_out=P)):
        assert call(L, **wrong) == BAD_ARGUMENT, wrong
    for other in (dict(page=12), dict(page=48), dict(width=1 << 27, page=16), dict(pages=1 << 27, page=16), dict(width=1, page=1 << 30, pages=2)):
        assert call(L, **other) == UNSUPPORTED, other


def test_cut_work(L):
    """An int per sequence, but for so few that one workgroup has them all."""
    for batch, width in ((1, 1), (64, 512), (8, 4096), (1, 1 << 15)):
        assert L.cubert_paged_cut_work(batch, width) == 0
    for batch, width in ((65, 1), (64, 513), (1, (1 << 15) + 1), (5000, 7)):
        assert L.cubert_paged_cut_work(batch, width) == batch
    assert L.cubert_paged_cut_work(0, 1 << 20) == 0


def test_extend_refuses(L):
    assert extend(L, rows=-1) == BAD_ARGUMENT
    assert extend(L, slots=None) == BAD_ARGUMENT
    assert extend(L, batch=1 << 16, rows=1 << 15) == UNSUPPORTED
    assert extend(L, batch=(1 << 18) + 1, rows=1) == UNSUPPORTED
    assert cut(L, batch=(1 << 18) + 1) == UNSUPPORTED
    assert extend(L, batch=LARGE, rows=0) == UNSUPPORTED
    assert extend(L, batch=LARGE, rows=LARGE) == UNSUPPORTED


def test_cut_refuses(L):
    assert cut(L, work=None, batch=65) == BAD_ARGUMENT
    assert cut(L, work=None, width=1 << 15) == BAD_ARGUMENT
    assert cut(L, batch=(1 << 25) + 1) == UNSUPPORTED


def pools(page_stride=None, head_stride=None, row_stride=None, pages=100, page=16, kv_heads=2, size=64):
    """Strides of [pages, kv_heads, page, size] one behind the other, unless others are given."""
    return (kv_heads * page * size if page_stride is None else page_stride, page * size if head_stride is None else head_stride,
            size if row_stride is None else row_stride, pages, page, kv_heads, size)


def write(L, t, k=P, v=P, ld=None, slots=P, tokens=5, k_pages=P, v_pages=P, **sizes):
    page_stride, head_stride, row_stride, pages, page, kv_heads, size = pools(**sizes)
    return getattr(L, "cubert_paged_write_" + t)(k, v, kv_heads * size if ld is None else ld, slots, tokens, k_pages, v_pages, page_stride,
                                                 head_stride, row_stride, pages, page, kv_heads, size, None)


# strides under which two elements share a place, or which no pool has
TOGETHER = (dict(page_stride=0), dict(head_stride=0), dict(row_stride=0), dict(row_stride=56), dict(page_stride=16 * 64), dict(page_stride=2048 - 8),
            dict(page_stride=-2048), dict(row_stride=128, head_stride=72), dict(head_stride=1 << 62), dict(page_stride=1 << 60))


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_write_refuses(L, t):
    for wrong in (dict(k=None), dict(v=None), dict(slots=None), dict(k_pages=None), dict(v_pages=None), dict(tokens=-1), dict(pages=0), dict(page=0),
                  dict(kv_heads=0), dict(size=0), dict(ld=127)) + TOGETHER:
        assert write(L, t, **wrong) == BAD_ARGUMENT, wrong
    for other in (dict(k=P + 8), dict(v=P + 8), dict(k_pages=P + 8), dict(v_pages=P + 8), dict(ld=130), dict(size=66), dict(page=24), dict(pages=1 << 27),
                  dict(page_stride=2050), dict(head_stride=1026, page_stride=4096), dict(row_stride=66, head_stride=2048, page_stride=4096),
                  dict(tokens=LARGE, kv_heads=64)):
        assert write(L, t, **other) == UNSUPPORTED, other
    assert write(L, t, tokens=0, k=None, slots=None) == 0


def attention(L, t, q=P, ldq=None, k=P, v=P, table=P, width=8, ld_table=None, lengths=P, ctx=P, ld_ctx=None, alpha=1.0, batch=2, heads=4, q_rows=3, left=-1,
              sinks=0, **sizes):
    page_stride, head_stride, row_stride, pages, page, kv_heads, size = pools(**sizes)
    return getattr(L, "cubert_attention_paged_" + t)(
        q, heads * size if ldq is None else ldq, k, v, page_stride, head_stride, row_stride, table, width, width if ld_table is None else ld_table,
        lengths, None, ctx, heads * size if ld_ctx is None else ld_ctx, alpha, batch, heads, kv_heads, q_rows, pages, page, size, left, sinks, None, 0,
        None)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_paged_refuses(L, t):
    for wrong in (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lengths=None), dict(ctx=None), dict(batch=-1), dict(heads=0),
                  dict(kv_heads=0), dict(kv_heads=3), dict(q_rows=-1), dict(q_rows=1 << 30), dict(pages=0), dict(page=0), dict(size=0), dict(sinks=-1),
                  dict(ldq=255), dict(ld_ctx=255), dict(width=0), dict(ld_table=7), dict(alpha=float("nan")), dict(alpha=float("inf")),
                  dict(alpha=float("-inf"))) + TOGETHER:
        assert attention(L, t, **wrong) == BAD_ARGUMENT, wrong
    for other in (dict(size=48), dict(size=256), dict(q=P + 8), dict(k=P + 8), dict(v=P + 8), dict(ctx=P + 8), dict(ldq=258), dict(ld_ctx=258),
                  dict(page=8), dict(page=1), dict(page=48), dict(width=1 << 26), dict(pages=1 << 27), dict(page_stride=2050),
                  dict(head_stride=1026, page_stride=4096), dict(row_stride=66, head_stride=2048, page_stride=4096), dict(batch=1 << 24), dict(batch=1 << 16, q_rows=1 << 16),
                  dict(row_stride=1 << 27, head_stride=64, page_stride=1 << 33)):
        assert attention(L, t, **other) == UNSUPPORTED, other
    assert attention(L, t, batch=0, q=None) == 0
    assert attention(L, t, q_rows=0, q=None) == 0


def test_attention_paged_partials_of_nothing(L):
    for half in (0, 1):
        for nothing in ((0, 4, 2, 1, 8, 16, 64), (1, 4, 3, 1, 8, 16, 64), (1, 4, 0, 1, 8, 16, 64), (1, 4, 2, 0, 8, 16, 64), (1, 4, 2, 1, 0, 16, 64),
                        (1, 4, 2, 1, 8, 0, 64), (1, 4, 2, 1, 8, 16, 0), (1 << 30, 1 << 20, 1 << 20, 1, 5000, 16, 64), (1, 4, 2, 1, LARGE, LARGE, 64),
                        (1, 4, 2, LARGE, 8, 16, 64)):
            assert L.cubert_attention_paged_partials(half, *nothing, -1, 0) == 0, nothing


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_wrappers_refuse_host_tensors():
    from cubert_amd import kernels
    pool, q = torch.zeros(4, 2, 16, 64), torch.zeros(1, 1, 4, 64)
    for call in (lambda: kernels.paged_extend(ints(2, 3), ints(2), ints(2), ints(9), ints(1), 16, 1),
                 lambda: kernels.paged_cut(ints(2, 3), ints(2), ints(2), ints(9), ints(1), 16),
                 lambda: kernels.paged_write(q[:, :, :2], q[:, :, :2], ints(1, 1), pool, pool),
                 lambda: kernels.attention_paged(q, pool, pool, ints(1, 3), ints(1))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_wrappers_refuse(monkeypatch):
    """Types, shapes and strides, before any call of the library."""
    from cubert_amd import kernels
    monkeypatch.setattr(kernels, "_device", lambda *tensors: 0)
    monkeypatch.setattr(kernels, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(kernels, "_run_on", lambda *args, **more: pytest.fail("called"))
    tables = (ints(2, 3), ints(2), ints(2), ints(9), ints(1), 16)
    for at, wrong in ((0, ints(2, 3).long()), (0, ints(6)), (0, ints(2, 0)), (0, ints(3, 2).t()), (0, ints(1, 3).expand(2, 3)), (1, ints(3)), (1, ints(2).long()),
                      (2, ints(1)), (2, ints(2).float()), (3, ints(9).long()), (3, ints(3, 3)), (3, ints(0)), (3, ints(18)[::2]), (4, ints(2)), (4, ints()),
                      (5, 0), (5, 12), (5, -16)):
        args = tables[:at] + (wrong,) + tables[at + 1:]
        with pytest.raises(ValueError):
            kernels.paged_extend(*args, 1)
        with pytest.raises(ValueError):
            kernels.paged_cut(*args)
    pool, q, n = torch.zeros(4, 2, 16, 64), torch.zeros(2, 3, 4, 64), ints(2)
    kv = q[:, :, :2]
    for call in (lambda: kernels.paged_write(kv.half(), kv, ints(2, 3), pool, pool), lambda: kernels.paged_write(kv, kv[:, :2], ints(2, 3), pool, pool),
                 lambda: kernels.paged_write(kv, kv, ints(2, 2), pool, pool), lambda: kernels.paged_write(kv, kv, ints(2, 3).long(), pool, pool),
                 lambda: kernels.paged_write(q, q, ints(2, 3), pool, pool), lambda: kernels.paged_write(kv, kv.contiguous(), ints(2, 3), pool, pool),
                 lambda: kernels.paged_write(kv, kv, ints(2, 3), pool, pool.half()), lambda: kernels.paged_write(kv, kv, ints(2, 3), pool, pool[:3]),
                 lambda: kernels.paged_write(kv, kv, ints(2, 3), pool, pool.transpose(1, 2).contiguous().transpose(1, 2)),
                 lambda: kernels.paged_write(kv, kv, ints(2, 3), pool[0], pool[0])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: kernels.attention_paged(q.half(), pool, pool, ints(2, 3), n), lambda: kernels.attention_paged(q, pool, pool, ints(3, 3), n),
                 lambda: kernels.attention_paged(q, pool, pool, ints(2, 3).long(), n), lambda: kernels.attention_paged(q, pool, pool, ints(2, 3), ints(3)),
                 lambda: kernels.attention_paged(q, pool, pool, ints(2, 3), n, first=ints(3)),
                 lambda: kernels.attention_paged(q, pool, pool, ints(2, 3), n, first=n.long()),
                 lambda: kernels.attention_paged(q[..., :32], pool, pool, ints(2, 3), n), lambda: kernels.attention_paged(q[:, :, ::2], pool, pool, ints(2, 3), n),
                 lambda: kernels.attention_paged(q[:, :, :3].contiguous(), pool, pool, ints(2, 3), n),
                 lambda: kernels.attention_paged(q, pool, pool[..., ::2], ints(2, 3), n), lambda: kernels.attention_paged(q[0], pool, pool, ints(2, 3), n)):
        with pytest.raises(ValueError):
            call()
    double = torch.zeros(4, 2, 16, 64, dtype=torch.float64)
    with pytest.raises(TypeError):
        kernels.attention_paged(q.double(), double, double, ints(2, 3), n)
    with pytest.raises(TypeError):
        kernels.paged_write(kv.double(), kv.double(), ints(2, 3), double, double)


def test_wrappers_refuse_what_32_bits_do_not_hold(monkeypatch):
    from cubert_amd import kernels
    monkeypatch.setattr(kernels, "_device", lambda *tensors: 0)
    large = (1 << 32) + 64

    def empty(*shape, dtype=torch.float16):
        return torch.empty(shape, dtype=dtype, device="meta")

    def whole(*shape):
        return empty(*shape, dtype=torch.int32)

    pool = empty(4, 2, 16, 64)
    for call in (lambda: kernels.paged_extend(whole(1, large), whole(1), None, whole(9), whole(1), 16, 1),
                 lambda: kernels.paged_extend(whole(1, 3), whole(1), None, whole(large), whole(1), 16, 1),
                 lambda: kernels.paged_extend(whole(1, 3), whole(1), None, whole(9), whole(1), 1 << 32, 1),
                 lambda: kernels.paged_extend(whole(1, 3), whole(1), None, whole(9), whole(1), 16, large),
                 lambda: kernels.paged_cut(whole(1, 3), whole(1), None, whole(9), whole(1), 16, large),
                 lambda: kernels.paged_cut(torch.empty_strided((2, 3), (large, 1), dtype=torch.int32, device="meta"), whole(2), None, whole(9), whole(1), 16),
                 lambda: kernels.paged_write(empty(1, large, 2, 64), empty(1, large, 2, 64), whole(1, large), pool, pool),
                 lambda: kernels.paged_write(empty(1, 1, 2, 64), empty(1, 1, 2, 64), whole(1, 1), empty(large, 2, 16, 64), empty(large, 2, 16, 64)),
                 lambda: kernels.attention_paged(empty(1, large, 4, 64), pool, pool, whole(1, 3), whole(1)),
                 lambda: kernels.attention_paged(empty(1, 1, 4, 64), pool, pool, whole(1, large), whole(1))):
        with pytest.raises(ValueError, match="2\\*\\*31"):
            call()


def test_bounds_of_any_size_reach_the_library(monkeypatch):
    from cubert_amd import kernels
    calls = []
    monkeypatch.setattr(kernels, "_device", lambda *tensors: 0)
    monkeypatch.setattr(kernels, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(kernels, "_run_on", lambda device, name, args: calls.append(args) or True)
    pool, q, n = torch.zeros(4, 2, 16, 64), torch.zeros(2, 3, 4, 64), ints(2)
    for left, sinks, sent in ((7, 4, (7, 4)), (-1, 0, (-1, 0)), (-(1 << 40), 0, (-1, 0)), (1 << 40, 1 << 40, (1 << 30, 1 << 30)), (5, -1, (5, -1)),
                              (5, 3 - (1 << 32), (5, -1))):
        kernels.attention_paged(q, pool, pool, ints(2, 3), n, left, sinks)
        assert calls[-1][-5:-3] == sent                    # left, sinks, partials, their number, stream


def test_tables_refuse_results_over_what_they_read(L):
    """Workgroups read lengths, counts and the stack when others write already."""
    ints = 4
    there = dict(table=1 << 20, lengths=2 << 20, counts=3 << 20, free=4 << 20, free_count=5 << 20, slots=6 << 20, lengths_out=7 << 20, free_out=8 << 20)
    count = dict(lengths=300, counts=300, free=100, free_count=1, slots=600, lengths_out=300, free_out=1)
    for out in ("slots", "lengths_out", "free_out"):
        for other in ("lengths", "counts", "free", "free_count", "slots", "lengths_out", "free_out"):
            if out == other:
                continue
            for at in {0, count[other] - 1, 1 - count[out]}:   # the same memory, the last of one the first of the other
                changed = dict(there)
                changed[out] = there[other] + ints * at
                assert extend(L, batch=300, rows=2, **changed) == BAD_ARGUMENT, (out, other, at)
    there["keep"], there["work"] = there.pop("counts"), there.pop("slots")
    count.update(keep=300, work=300)
    for out in ("work", "lengths_out", "free_out"):
        for other in ("lengths", "keep", "free", "free_count", "work", "lengths_out", "free_out"):
            if out == other:
                continue
            for at in {0, count[other] - 1, 1 - count[out]}:
                if (out, other, at) == ("lengths_out", "keep", 0):  # (which works: what is written is what was read, within its range)
                    continue
                changed = dict(there)
                changed[out] = there[other] + ints * at
                assert cut(L, batch=300, **changed) == BAD_ARGUMENT, (out, other, at)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_write_refuses_one_pool_for_both(L, t):
    assert write(L, t, k_pages=Q, v_pages=Q) == BAD_ARGUMENT
