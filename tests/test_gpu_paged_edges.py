"""Paged attention where its number formats end: keys and queries of very different
sizes, scores far past what an fp32 exponent resolves. Both forms of the kernel, against
64-bit attention within the bound that paged_ref derives."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import paged_ref as R  # noqa: E402
from tests.test_gpu_paged import check_attention, gen, randn  # noqa: E402


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    assert mlb.paged_attention_status() == (0, 0)


def stored(seqs, k, v):
    """A cache that holds k and v, and the values its codes stand for."""
    cache = mlb.CudaPagedKvCache(1, seqs.n_pages, seqs.page, k.shape[1], k.shape[2])
    cache.AppendDevice(0, k, v, *seqs.whole(), rope_type=mlb.ROPE_NONE)
    return (cache, *cache.ReadDevice(0, *seqs.whole(), seqs.total))


# rows of a call whose 8 heads over 2 KV heads take the decode form (1, 6) or the prompt form
ROWS = [1, 6, 1200]


def both_forms(n, dtype):
    assert R.prompt_form(n, 1, 2, 4, dtype) == (n == 1200)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 1e-6, 5e4])
def test_keys_of_any_size(cuda, size, n, dtype):
    """Queries are as large as keys are small, so that scores stay ordinary."""
    dtype = getattr(torch, dtype)
    both_forms(n, dtype)
    seqs = R.Seqs([n], [1300], 32, seed=n)
    g = gen(51)
    cache, kk, vv = stored(seqs, randn(g, 1300, 2, 128) * size, randn(g, 1300, 2, 128))
    q = (randn(g, n, 8, 128) * (2 / size)).to(dtype)
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, 128)
    check_attention(out, q, kk, vv, seqs, 128, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("sizes", [(1e-2, 1e-3, 1e-4, 1e-5), (3e4, 3e3, 6e4, 5e2)])
def test_keys_of_many_sizes_in_one_sequence(cuda, sizes, n, dtype):
    """A token has keys in one of four groups of 32 dimensions, each group's of another
    size and its queries to match: every score is ordinary whichever the token's size,
    within a tile of tokens and within 16 neighbours."""
    dtype = getattr(torch, dtype)
    seqs = R.Seqs([n], [1300], 32, seed=n)
    g = gen(52)
    k = randn(g, 1300, 2, 4, 32)
    group = torch.randint(4, (1300,), device="cuda", generator=g)
    k *= torch.nn.functional.one_hot(group, 4)[:, None, :, None]
    each = torch.tensor(sizes, device="cuda")[:, None]
    cache, kk, vv = stored(seqs, (k * each).flatten(2), randn(g, 1300, 2, 128))
    q = (randn(g, n, 8, 4, 32) * 4 / each).flatten(2).to(dtype)
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, 128)
    check_attention(out, q, kk, vv, seqs, 128, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("size", [1e3, 1e5, 1e7, 1e8, 3e9, 1e12, 1e25])
def test_scores_of_any_size(cuda, size, n, dtype):
    """A query is one dimension, so a score is one product, exact in fp32, and equal
    keys tie exactly. Scores of unlike keys are hundreds apart or more: a row is the
    mean of the values whose keys tie at the top, whatever the scores' size."""
    dtype = getattr(torch, dtype)
    both_forms(n, dtype)
    hd, length = 64, 1300
    seqs = R.Seqs([n], [length], 32, seed=n)
    g = gen(53)
    # keys of one scale (7 in every block), so integers, each token with its twin
    k = torch.randint(-5, 6, (length // 2, 2, hd), device="cuda", generator=g).float()
    k[:, :, 1::32] = 7.0
    top = torch.rand(length // 2, device="cuda", generator=g) < 0.01
    k[:, :, 0] = torch.where(top[:, None], 7.0, k[:, :, 0])
    k = k.repeat(2, 1, 1)
    cache, kk, vv = stored(seqs, k, randn(g, length, 2, hd))
    assert torch.equal(kk, k)
    q = torch.zeros(n, 8, hd, device="cuda")
    q[:, :, 0] = (1 + torch.rand(n, 8, device="cuda", generator=g)) * size
    q[:, ::3, 0] *= -1
    q = q.bfloat16().to(dtype)
    scale = 1.7
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, hd, scale=scale)
    want, vabs, (_, vmax) = R.attention(q, kk, vv, length, n, scale)
    # scores bring no error: neither the tied ones' differences, 0, nor the others' p, 0
    none = torch.zeros(n, 8, 1, dtype=torch.float64)
    tol = R.attention_bound(want, vabs, (none, vmax), length, dtype, n == 1200)
    err = (out.double().cpu() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"error {err.max():.3e}, worst ratio {(err / tol).max():.2f}"


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("size,scale", [(1e6, 0.1), (1e9, 0.1), (1.0, 1e10), (1e30, 1e-20)])
def test_outputs_stay_within_the_values(cuda, size, scale, n, dtype):
    """Whatever the scores, a row's result is a mean of the values that it sees."""
    dtype = getattr(torch, dtype)
    hd, length = 128, 1300
    seqs = R.Seqs([n], [length], 32, seed=n)
    g = gen(54)
    cache, _, vv = stored(seqs, randn(g, length, 2, hd), randn(g, length, 2, hd))
    q = (randn(g, n, 8, hd) * size).to(dtype)
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, hd, scale=scale)
    low, high = (getattr(vv, f)(0)[None].repeat_interleave(4, 1) for f in ("amin", "amax"))
    # P and V are rounded to fp16 at worst, the sum cut once per 16 tokens, the result
    # rounded to its type
    slack = vv.abs().max() * (2.0 ** -11 + 2.0 ** -11 + 82 * 2.0 ** -23 + 2.0 ** -8)
    assert (out >= low - slack).all() and (out <= high + slack).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", ROWS[1:])
def test_rows_that_are_no_numbers_keep_to_themselves(cuda, n, dtype):
    """Infinite and NaN queries: the call ends, and other rows are what they were."""
    dtype = getattr(torch, dtype)
    hd, length = 128, 1300
    seqs = R.Seqs([n], [length], 32, seed=n)
    g = gen(55)
    cache, kk, vv = stored(seqs, randn(g, length, 2, hd), randn(g, length, 2, hd))
    q = randn(g, n, 8, hd, dtype=dtype)
    want, vabs, top = R.attention(q, kk, vv, length, n, 0.1)
    good = torch.ones(n, 8, dtype=torch.bool)
    for row, head, dim, x in ((0, 0, 3, "inf"), (2, 1, 127, "-inf"), (n - 1, 7, 0, "nan"),
                              (n // 2, 4, slice(None), "inf"), (n // 2, 5, slice(None), "nan")):
        q[row, head, dim] = float(x)
        good[row, head] = False
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, hd, scale=0.1)
    tol = R.attention_bound(want, vabs, top, length, dtype, n == 1200)
    err = (out.double().cpu() - want).abs()
    assert (err <= tol)[good].all()
    assert not torch.isfinite(out.cpu()[~good]).any()


BOTTOM, TOP = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [5, 4800])
@pytest.mark.parametrize("offsets", [
    (0, 3, TOP, -2, 5), (TOP, BOTTOM, TOP, -1, TOP), (-5, 2, BOTTOM, TOP, 3), (9, 7, 7, -1, -2)])
@pytest.mark.parametrize("lens", [(40, 41, 42, 43), (BOTTOM, TOP, -1, 0)])
@pytest.mark.parametrize("width", [3, 48])
def test_offsets_and_lengths_of_any_value(cuda, width, lens, offsets, n, dtype):
    """Nothing past the call's rows is written, whatever the arrays hold."""
    dtype = getattr(torch, dtype)
    kv, hd, page, heads = 2, 32, 16, 8
    assert R.prompt_form(n, 4, kv, heads // kv, dtype) == (n > 5)
    i32 = dict(dtype=torch.int32, device="cuda")
    where = (torch.tensor(offsets, **i32), torch.tensor(lens, **i32),
             (torch.arange(4 * width, **i32) % 16).view(4, width))  # 12 .. 15: not in the pool
    g = gen(56)
    q, k, v = (randn(g, n, h, hd, dtype=dtype) for h in (heads, kv, kv))
    cache = mlb.CudaPagedKvCache(3, 12, page, kv, hd)
    cache.pages.fill_(85)
    cache.pages[1] = 0
    wide = torch.full((n + 64, heads, hd), 3.0, dtype=dtype, device="cuda")
    out = wide[32:32 + n]
    mlb.CudaPagedAttentionDeviceInput(q, cache, 1, *where, heads, kv, hd, out=out)
    cache.AppendDevice(1, k, v, *where, q=q, q_out=out)
    for x in cache.ReadDevice(1, *where, n):
        assert torch.isfinite(x).all()
    assert (wide[:32] == 3).all() and (wide[32 + n:] == 3).all()
    assert (cache.pages[0] == 85).all() and (cache.pages[2] == 85).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_a_wait_that_gives_up_is_told(cuda, bf16):
    """A barrier that never completes: every role of the prompt form gives up, the
    status word says so once, no row keeps what the buffer held, and the next call on
    the device is right."""
    code, where, rows = mlb.paged_attention_wait_selftest(bf16)
    assert code == mlb.ERR_TIMEOUT and 1001 <= where <= 1011 and rows == 8
    assert mlb.paged_attention_status() == (0, 0)
    test_keys_of_any_size(cuda, 1.0, 1200, "bfloat16" if bf16 else "float32")


@pytest.mark.parametrize("n", ROWS)
def test_queries_and_outputs_side_by_side(cuda, n):
    """Rows of one buffer in turn: not an overlap, and what separate buffers give."""
    seqs = R.Seqs([n], [1300], 32, seed=n)
    g = gen(57)
    cache, _, _ = stored(seqs, randn(g, 1300, 2, 64), randn(g, 1300, 2, 64))
    both = randn(g, n, 16, 64)
    q, out = both[:, :8], both[:, 8:]
    want = mlb.CudaPagedAttentionDeviceInput(q.clone(), cache, 0, *seqs.where(), 8, 2, 64)
    mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, 64, out=out)
    assert torch.equal(out, want)
    with pytest.raises(mlb.MlbError, match="must not overlap"):
        mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, 64,
                                          out=both[:, 1:9])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [1, 7, 1500])
def test_append_in_one_buffer(cuda, n, dtype):
    """q, k and v cut out of one projection's rows, q rotated in place or into the same
    rows' spare part: what separate buffers give, k and v left as they were."""
    dtype = getattr(torch, dtype)
    seqs = R.Seqs([n], [n + 9], 32, seed=n)
    g = gen(58)
    fused = randn(g, n, 8 + 2 + 2 + 8, 64, dtype=dtype)
    caches = [mlb.CudaPagedKvCache(1, seqs.n_pages, 32, 2, 64) for _ in range(3)]
    want = caches[0].AppendDevice(0, fused[:, 8:10].clone(), fused[:, 10:12].clone(),
                                  *seqs.where(), q=fused[:, :8].clone())
    for cache, at in ((caches[1], 0), (caches[2], 12)):
        x = fused.clone()
        q, k, v = x[:, :8], x[:, 8:10], x[:, 10:12]
        out = cache.AppendDevice(0, k, v, *seqs.where(), q=q, q_out=x[:, at:at + 8])
        assert torch.equal(out, want) and torch.equal(cache.pages, caches[0].pages)
        assert torch.equal(x[:, 8:12], fused[:, 8:12])
        with pytest.raises(mlb.MlbError, match="q_out must not overlap k or v"):
            cache.AppendDevice(0, k, v, *seqs.where(), q=fused[:, :8], q_out=x[:, 9:17])
        with pytest.raises(mlb.MlbError, match="q_out must be q itself or not overlap it"):
            cache.AppendDevice(0, k, v, *seqs.where(), q=x[:, 12:20], q_out=x[:, 11:19])
