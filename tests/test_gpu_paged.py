"""The paged Q4_0 KV cache and its attention on the GPU, against 64-bit forms.

Codes are compared bit for bit with the host quantiser; rotated queries within
half a step of their type; attention within the bound that paged_ref derives.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import paged_ref as R  # noqa: E402

ROPE = {"normal": mlb.ROPE_NORMAL, "neox": mlb.ROPE_NEOX}


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    assert mlb.paged_attention_status() == (0, 0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def filled(seqs, kv, hd, seed, layers=1, layer=0, pool=None):
    """A cache that holds random keys and values of whole sequences, and the
    values its codes stand for, [total, kv, hd] each."""
    g = gen(seed)
    cache = mlb.CudaPagedKvCache(layers, seqs.n_pages, seqs.page, kv, hd)
    if pool is not None:
        cache.pages.fill_(pool)
    k, v = randn(g, seqs.total, kv, hd), randn(g, seqs.total, kv, hd)
    cache.AppendDevice(layer, k, v, *seqs.whole(), rope_type=mlb.ROPE_NONE)
    kk, vv = cache.ReadDevice(layer, *seqs.whole(), seqs.total)
    return cache, kk, vv


def check_attention(out, q, kk, vv, seqs, hd, dtype, scale=None):
    scale = 1 / math.sqrt(hd) if scale is None else scale
    row = at = 0
    kv = kk.shape[1]
    prompt = R.prompt_form(seqs.rows, len(seqs.new), kv, q.shape[1] // kv, dtype)
    for n, length in zip(seqs.new, seqs.lens):
        if n:
            m = min(n, length)  # rows before position 0 see nothing
            dead = out[row:row + n - m]
            assert (dead == 0).all()
            want, vabs, top = R.attention(q[row + n - m:row + n], kk[at:at + length],
                                          vv[at:at + length], length, m, scale)
            got = out[row + n - m:row + n].double().cpu()
            err, tol = (got - want).abs(), R.attention_bound(want, vabs, top, length, dtype,
                                                                      prompt)
            assert torch.isfinite(got).all()
            assert (err <= tol).all(), f"error {err.max():.3e}, worst ratio {(err / tol).max():.2f}"
        row, at = row + n, at + length


@pytest.mark.parametrize("kv,hd,page,rope,dtype", [
    (8, 128, 16, "normal", "float32"), (8, 128, 64, "neox", "bfloat16"),
    (6, 48, 16, "normal", "float32"), (6, 48, 32, "neox", "float32"),
    (2, 64, 48, "neox", "float32"), (3, 8, 16, "normal", "bfloat16"),
    (1, 40, 128, "neox", "bfloat16"), (4, 96, 32, "normal", "float32"),
    (2, 32, 16, "neox", "float32")])
def test_append_rotates_and_quantises(cuda, kv, hd, page, rope, dtype):
    dtype = getattr(torch, dtype)
    seqs = R.Seqs([1, 5, 0, 17, 3], [1, 300, 40, 17, 100003], page, seed=kv + hd)
    g = gen(hd)
    heads = 2 * kv
    q = randn(g, seqs.rows, heads, hd, dtype=dtype)
    k = randn(g, seqs.rows, kv, hd, dtype=dtype) * 3
    v = randn(g, seqs.rows, kv, hd, dtype=dtype)
    v[0, 0] = 0  # a block of zeros
    v[1, 0] *= 1e-6  # scales below fp16's normal range
    cache = mlb.CudaPagedKvCache(2, seqs.n_pages, page, kv, hd)
    before = cache.pages.clone()
    theta = 500000.0
    q_out = cache.AppendDevice(1, k, v, *seqs.where(), theta=theta, rope_type=ROPE[rope], q=q)
    kk, vv = cache.ReadDevice(1, *seqs.where(), seqs.rows)
    neox = rope == "neox"
    assert torch.equal(vv.double().cpu(), R.quantise(v.float()))
    assert torch.equal(kk.double().cpu(), R.quantise(R.rotate(k, seqs.pos, theta, neox).float()))
    want = R.rotate(q, seqs.pos, theta, neox)
    # rounded to fp32, then to the type; angles themselves to 2^-53 of 1e5 radians
    tol = want.abs() * (2.0 ** -24 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) + 1e-10
    assert ((q_out.double().cpu() - want).abs() <= tol).all()
    # nothing else was written: the other layer, and pages no sequence owns
    assert torch.equal(cache.pages[0], before[0])
    for p in seqs.spare:
        assert torch.equal(cache.pages[1, p], before[1, p])
    # in place
    q2 = q.clone()
    cache.AppendDevice(1, k, v, *seqs.where(), theta=theta, rope_type=ROPE[rope], q=q2, q_out=q2)
    assert torch.equal(q2, q_out)


def test_append_one_token_at_a_time_is_the_same_cache(cuda):
    kv, hd, page, length = 2, 128, 16, 37
    seqs = R.Seqs([length], [length], page, seed=3)
    g = gen(1)
    k, v = randn(g, length, kv, hd), randn(g, length, kv, hd)
    whole = mlb.CudaPagedKvCache(1, seqs.n_pages, page, kv, hd)
    whole.AppendDevice(0, k, v, *seqs.where())
    one = mlb.CudaPagedKvCache(1, seqs.n_pages, page, kv, hd)
    offs = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for t in range(length):
        n = torch.tensor([t + 1], dtype=torch.int32, device="cuda")
        one.AppendDevice(0, k[t:t + 1], v[t:t + 1], offs, n, seqs.table)
    assert torch.equal(one.pages, whole.pages)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rope", ["normal", "neox", "none"])
@pytest.mark.parametrize("heads,kv,hd", [(5, 2, 128), (3, 3, 40), (7, 1, 8), (2, 3, 96),
                                         (6, 6, 48)])
def test_append_of_many_rows_is_that_of_few(cuda, heads, kv, hd, rope, dtype):
    """More rows than 8 per SM go another way: the same bits as in calls of 400,
    rows of no position among them."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n, page = 8 * sms + 37, 32
    seqs = R.Seqs([n], [n - 3], page, seed=heads)  # three rows are before position 0
    g = gen(hd)
    dtype = getattr(torch, dtype)
    rope = {**ROPE, "none": mlb.ROPE_NONE}[rope]
    rows = n + 5  # and five behind the last sequence
    q, k, v = (randn(g, rows, h, hd, dtype=dtype) for h in (heads, kv, kv))
    table = seqs.table.clone()
    table[0, 3] = seqs.n_pages  # not in the pool
    many, few = (mlb.CudaPagedKvCache(1, seqs.n_pages, page, kv, hd) for _ in range(2))
    out = torch.full_like(q, 7.0)
    many.AppendDevice(0, k, v, seqs.offsets, seqs.seq_lens, table, rope_type=rope, q=q, q_out=out)
    assert (out[:3] == 7).all() and (out[n:] == 7).all()
    i32 = dict(dtype=torch.int32, device="cuda")
    for r in range(0, n, 400):
        e = min(r + 400, n)
        part = few.AppendDevice(0, k[r:e], v[r:e], torch.tensor([0, e - r], **i32),
                                torch.tensor([e - 3], **i32), table, rope_type=rope, q=q[r:e])
        first = 3 if r == 0 else 0
        assert torch.equal(out[r + first:e], part[first:])
    assert torch.equal(many.pages, few.pages)


def test_rows_that_belong_to_no_position_are_left_alone(cuda):
    """Rows behind the last sequence, at negative positions, past the table and
    on pages outside the pool."""
    kv, hd, page = 2, 64, 16
    seqs = R.Seqs([3, 4, 2], [10, 20, 33], page, seed=5)
    g = gen(2)
    rows = seqs.rows + 4  # four rows of padding
    q, k, v = (randn(g, rows, h, hd) for h in (4, kv, kv))
    cache = mlb.CudaPagedKvCache(1, seqs.n_pages, page, kv, hd)
    lens = seqs.seq_lens.clone()
    lens[0] = 2  # three rows end at length 2: the first is at position -1
    table = seqs.table.clone()
    table[1, 1] = seqs.n_pages  # positions 16..19 of sequence 1
    table[2, 1] = -1  # positions 16..31 of sequence 2
    lens[2] = 33
    q_out = torch.full_like(q, 7.0)
    before = cache.pages.clone()
    cache.AppendDevice(0, k, v, seqs.offsets, lens, table, q=q, q_out=q_out,
                       rope_type=mlb.ROPE_NONE)
    assert (q_out[seqs.rows:] == 7).all() and (q_out[0] == 7).all()
    assert torch.equal(q_out[1:seqs.rows], q[1:seqs.rows])
    kk, _ = cache.ReadDevice(0, seqs.offsets, lens, table, rows)
    want = R.quantise(k).float().cuda()
    # row: 0 at -1; 3..6 at 16..19 (no page); 7 at 31 (no page); 8 at 32
    for r in range(rows):
        if r in (1, 2, 8):
            assert torch.equal(kk[r], want[r]), r
        else:
            assert (kk[r] == 0).all(), r
    touched = {int(table[0, 0]), int(table[2, 2])}
    for p in range(seqs.n_pages):
        assert torch.equal(cache.pages[0, p], before[0, p]) == (p not in touched)
    # past the table's last column: nothing is stored, nothing read
    far = torch.tensor([10 ** 9, 20, 33], dtype=torch.int32, device="cuda")
    before = cache.pages.clone()
    offs = torch.tensor([0, 3, 3, 3], dtype=torch.int32, device="cuda")
    cache.AppendDevice(0, k[:3], v[:3], offs, far, table)
    assert torch.equal(cache.pages, before)


SHAPES = [  # heads, kv, hd, page
    (32, 8, 128, 16), (64, 8, 128, 64), (4, 4, 128, 32), (6, 6, 48, 16), (8, 2, 64, 48),
    (12, 4, 96, 128), (16, 1, 128, 32), (7, 7, 40, 16), (4, 2, 32, 16), (10, 2, 8, 16),
    (24, 2, 64, 16)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_decode_attention(cuda, heads, kv, hd, page, dtype):
    """One row per sequence, lengths around every boundary."""
    dtype = getattr(torch, dtype)
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 500, 1, 777]
    new = [1] * len(lens)
    new[4] = 0  # a sequence without a row
    seqs = R.Seqs(new, lens, page, seed=heads)
    cache, kk, vv = filled(seqs, kv, hd, heads + hd, pool=255)
    q = randn(gen(9), seqs.rows, heads, hd, dtype=dtype) * 2
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd)
    check_attention(out, q, kk, vv, seqs, hd, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_ragged_rows_attention(cuda, heads, kv, hd, page, dtype):
    """Several rows per sequence, causal, some before the first position."""
    dtype = getattr(torch, dtype)
    new, lens = [3, 0, 40, 1, 9, 130, 5, 70], [3, 9, 40, 200, 300, 131, 2, 600]
    seqs = R.Seqs(new, lens, page, seed=heads + 1)
    cache, kk, vv = filled(seqs, kv, hd, heads + hd, layers=2, layer=1, pool=255)
    q = randn(gen(11), seqs.rows, heads, hd, dtype=dtype) * 2
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 1, *seqs.where(), heads, kv, hd,
                                            scale=0.11)
    check_attention(out, q, kk, vv, seqs, hd, dtype, scale=0.11)


@pytest.mark.parametrize("new,lens,heads,kv,dtype", [
    ([1], [9001], 32, 8, "float32"), ([1], [30000], 16, 1, "bfloat16"),
    ([2, 1], [12000, 5], 8, 8, "float32"), ([300], [1500], 8, 2, "bfloat16"),
    ([300], [1500], 8, 2, "float32"), ([1] * 70, list(range(1, 71)), 16, 2, "float32")])
def test_long_and_many(cuda, new, lens, heads, kv, dtype):
    """Units that many CTAs share, and more sequences than a block has threads'
    worth of work to scan at once."""
    dtype = getattr(torch, dtype)
    seqs = R.Seqs(new, lens, 64, seed=1)
    cache, kk, vv = filled(seqs, kv, 128, 77)
    q = randn(gen(13), seqs.rows, heads, 128, dtype=dtype) * 3
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, 128)
    check_attention(out, q, kk, vv, seqs, 128, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,lens,heads,kv,hd", [
    ([600], [600], 32, 8, 128), ([300, 200, 7, 0, 130], [300, 333, 900, 4, 128], 32, 16, 128),
    ([257] * 6, [257, 300, 640, 257, 1000, 200], 24, 24, 96),
    ([128] * 20, [128 + 37 * i for i in range(20)], 16, 8, 64), ([1000], [1000], 40, 40, 40),
    ([90] * 40, [90] * 40, 16, 4, 32)])
def test_prompts(cuda, new, lens, heads, kv, hd, dtype):
    """Calls that take the prompt form: row tiles that end inside a token, tiles whose
    second half is empty, lengths on both sides of its steps, more rows than length."""
    dtype = getattr(torch, dtype)
    seqs = R.Seqs(new, lens, 32, seed=len(new))
    assert R.prompt_form(seqs.rows, len(new), kv, heads // kv, dtype)
    cache, kk, vv = filled(seqs, kv, hd, 19, pool=255)
    q = randn(gen(23), seqs.rows, heads, hd, dtype=dtype) * 2
    q[0] *= 30  # scores that rise by far more than a step allows for
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd)
    check_attention(out, q, kk, vv, seqs, hd, dtype)
    again = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (6, 6, 48), (4, 4, 96), (10, 2, 8)])
@pytest.mark.parametrize("rows", [1, 5, 20])
def test_short_tables(cuda, rows, heads, kv, hd, dtype):
    """Tables of at most 256 or 512 tokens keep units whole; wider ones do not."""
    dtype = getattr(torch, dtype)
    for lens in ([5, 1, 250, 256, 16, 130, 20], [500, 37, 512] + list(range(20, 490, 13))):
        seqs = R.Seqs([rows] * len(lens), lens, 16, seed=rows)
        cache, kk, vv = filled(seqs, kv, hd, heads, pool=255)
        q = randn(gen(hd), seqs.rows, heads, hd, dtype=dtype)
        wide = torch.cat((seqs.table, torch.full_like(seqs.table, -1)), 1)
        for table in (seqs.table, wide):
            out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, seqs.seq_lens,
                                                    table, heads, kv, hd)
            check_attention(out, q, kk, vv, seqs, hd, dtype)


def test_many_sequences(cuda):
    lens = [1 + (i * 37) % 90 for i in range(400)]
    new = [(i % 5 != 3) * 1 for i in range(400)]
    seqs = R.Seqs(new, lens, 16, seed=2)
    cache, kk, vv = filled(seqs, 2, 32, 5)
    q = randn(gen(3), seqs.rows, 4, 32)
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 4, 2, 32)
    check_attention(out, q, kk, vv, seqs, 32, torch.float32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_small_scales_keep_their_precision(cuda, dtype):
    """Keys and values of very different sizes along the sequence."""
    dtype = getattr(torch, dtype)
    kv, hd, length, n = 2, 128, 700, 40
    seqs = R.Seqs([n], [length], 32, seed=9)
    g = gen(21)
    k, v = randn(g, length, kv, hd), randn(g, length, kv, hd)
    v *= torch.logspace(-6, 3, length, device="cuda")[torch.randperm(length, device="cuda",
                                                                     generator=g)][:, None, None]
    v[:, 1] *= 1e-4
    cache = mlb.CudaPagedKvCache(1, seqs.n_pages, 32, kv, hd)
    cache.AppendDevice(0, k, v, *seqs.whole(), rope_type=mlb.ROPE_NONE)
    kk, vv = cache.ReadDevice(0, *seqs.whole(), length)
    for rows in (1, n):
        s = R.Seqs([rows], [length], 32, seed=9)
        q = randn(g, rows, 8, hd, dtype=dtype)
        q[0, 0] *= 1e-20
        q[0, 1] *= 1e3
        out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *s.where(), 8, kv, hd)
        check_attention(out, q, kk, vv, s, hd, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [1, 6, 90, 700])
def test_what_a_row_does_not_see_has_no_say(cuda, n, dtype):
    """Infinite and NaN values past a row, and in pages and slots of no one."""
    dtype = getattr(torch, dtype)
    kv, hd, page, heads = 2, 64, 32, 8
    length = 200 if n < 200 else 750
    seqs = R.Seqs([n], [length], page, seed=4)
    g = gen(6)
    k, v = randn(g, length, kv, hd), randn(g, length, kv, hd)
    q = randn(g, n, heads, hd, dtype=dtype)
    outs = []
    for bad in (False, True):
        cache = mlb.CudaPagedKvCache(1, seqs.n_pages, page, kv, hd)
        cache.pages.fill_(255 if bad else 0)
        k2, v2 = k.clone(), v.clone()
        if bad and n > 1:
            k2[-1], v2[-1] = math.nan, math.inf  # the last row's own token
            v2[-2, :, ::3] = -math.inf
        cache.AppendDevice(0, k2, v2, *seqs.whole(), rope_type=mlb.ROPE_NONE)
        outs.append(mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd))
    kk, vv = cache.ReadDevice(0, *seqs.whole(), length)
    if n == 1:
        assert torch.equal(outs[0], outs[1])
    else:
        # rows before the last two never see them; an infinite scale in a tile
        # only costs the tile's exponent range
        a, b = outs[0][:n - 2].double(), outs[1][:n - 2].double()
        assert torch.isfinite(b).all()
        assert ((a - b).abs() <= a.abs().max() * (2.0 ** -7 if dtype == torch.bfloat16
                                                 else 2.0 ** -16)).all()


def test_pages_outside_the_pool_are_not_seen(cuda):
    kv, hd, page, heads = 2, 128, 16, 8
    for n, dtype in ((1, torch.float32), (3, torch.bfloat16), (64, torch.float32),
                     (1100, torch.float32), (1100, torch.bfloat16)):
        length = max(300, n)
        seqs = R.Seqs([n], [length], page, seed=8)
        cache, kk, vv = filled(seqs, kv, hd, 4)
        q = randn(gen(5), n, heads, hd, dtype=dtype)
        table = seqs.table.clone()
        table[0, 2] = -5
        table[0, 3] = seqs.n_pages
        table[0, 11] = 2 ** 31 - 1
        absent = [t for t in range(length) if t // page in (2, 3, 11)]
        out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, seqs.seq_lens, table,
                                                heads, kv, hd)
        want, vabs, top = R.attention(q, kk, vv, length, n, 1 / math.sqrt(hd), absent)
        err = (out.double().cpu() - want).abs()
        prompt = R.prompt_form(n, 1, kv, heads // kv, dtype)
        assert (err <= R.attention_bound(want, vabs, top, length, dtype, prompt)).all()
        none = torch.full_like(table, -1)
        out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, seqs.seq_lens, none,
                                                heads, kv, hd)
        assert (out == 0).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [1, 20, 1200])
def test_first_pages_missing(cuda, n, dtype):
    """Rows whose first sight of the cache comes late, at scores far below zero."""
    dtype = getattr(torch, dtype)
    kv, hd, page, heads, length = 2, 64, 16, 8, 1300
    seqs = R.Seqs([n], [length], page, seed=8)
    g = gen(14)
    cache = mlb.CudaPagedKvCache(1, seqs.n_pages, page, kv, hd)
    k, v = randn(g, length, kv, hd) * 0.3 + 1.0, randn(g, length, kv, hd)
    cache.AppendDevice(0, k, v, *seqs.whole(), rope_type=mlb.ROPE_NONE)
    kk, vv = cache.ReadDevice(0, *seqs.whole(), length)
    q = (randn(g, n, heads, hd) - 25.0).to(dtype)  # scores near -200
    table = seqs.table.clone()
    table[0, :30] = -1
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, seqs.seq_lens, table, heads,
                                            kv, hd)
    absent = list(range(30 * page))
    want, vabs, top = R.attention(q, kk, vv, length, n, 1 / math.sqrt(hd), absent)
    prompt = R.prompt_form(n, 1, kv, heads // kv, dtype)
    err = (out.double().cpu() - want).abs()
    assert (err <= R.attention_bound(want, vabs, top, length, dtype, prompt)).all()
    assert n == 1 or (out[:max(0, n - (length - 30 * page))] == 0).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,over", [(1, 1), (9, 4), (9, 40), (1200, 700)])
def test_lengths_past_the_page_table(cuda, n, over, dtype):
    """Rows keep their positions when the sequence has outgrown its table: they
    see what the table holds up to their own."""
    dtype = getattr(torch, dtype)
    heads, kv, hd, page, held = 32, 4, 64, 32, 1600
    seqs = R.Seqs([n], [held], page, seed=n)
    cache, kk, vv = filled(seqs, kv, hd, over)
    q = randn(gen(n), n, heads, hd, dtype=dtype)
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, seqs.seq_lens + over,
                                            seqs.table, heads, kv, hd)
    more = torch.zeros(over, kv, hd, device="cuda")
    length = held + over
    want, vabs, top = R.attention(q, torch.cat((kk, more)), torch.cat((vv, more)), length, n,
                                  1 / math.sqrt(hd), absent=range(held, length))
    prompt = R.prompt_form(n, 1, kv, heads // kv, dtype)
    err = (out.double().cpu() - want).abs()
    tol = R.attention_bound(want, vabs, top, length, dtype, prompt)
    assert (err <= tol).all(), f"error {err.max():.3e}, worst ratio {(err / tol).max():.2f}"


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_and_unaligned_rows(cuda, dtype):
    """Rows cut out of one projection's output, and at odd addresses."""
    dtype = getattr(torch, dtype)
    heads, kv, hd = 8, 2, 64
    seqs = R.Seqs([4, 1, 30], [50, 7, 90], 16, seed=6)
    g = gen(31)
    fused = randn(g, seqs.rows, (heads + 2 * kv) * hd, dtype=dtype)
    q = fused[:, :heads * hd].unflatten(1, (heads, hd))
    k = fused[:, heads * hd:(heads + kv) * hd].unflatten(1, (kv, hd))
    v = fused[:, (heads + kv) * hd:].unflatten(1, (kv, hd))
    odd = torch.empty(fused.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(fused)
    odd.copy_(fused)
    qo, ko, vo = (odd[:, a * hd:b * hd].unflatten(1, (b - a, hd))
                  for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    res = []
    for qq, kk, vv in ((q.contiguous(), k.contiguous(), v.contiguous()), (q, k, v), (qo, ko, vo)):
        cache = mlb.CudaPagedKvCache(1, seqs.n_pages, 16, kv, hd)
        r = cache.AppendDevice(0, kk, vv, *seqs.where(), q=qq)
        o = mlb.CudaPagedAttentionDeviceInput(qq, cache, 0, *seqs.where(), heads, kv, hd)
        res.append((r, cache.pages, o))
    for other in res[1:]:
        for a, b in zip(res[0], other):
            assert torch.equal(a, b)
    # into a strided output
    wide = torch.full((seqs.rows, heads + 3, hd), 5.0, dtype=dtype, device="cuda")
    o = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd,
                                          out=wide[:, :heads])
    assert torch.equal(o, res[0][2]) and (wide[:, heads:] == 5).all()


def test_rows_behind_the_last_sequence_are_left_alone(cuda):
    heads, kv, hd = 8, 2, 64
    for new in ([1, 1], [40, 3]):
        seqs = R.Seqs(new, [100, 50], 16, seed=6)
        cache, _, _ = filled(seqs, kv, hd, 1)
        rows = seqs.rows + 5
        q = randn(gen(1), rows, heads, hd)
        out = torch.full_like(q, 3.0)
        mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd, out=out)
        assert (out[seqs.rows:] == 3).all() and (out[:seqs.rows] != 3).any()


@pytest.mark.parametrize("n,dtype", [(1, "float32"), (3, "bfloat16"), (900, "bfloat16"),
                                     (900, "float32")])
def test_graph_replay_with_new_lengths(cuda, n, dtype):
    """A captured step follows the lengths and tables that its buffers hold when
    it is replayed, on another stream, and twice gives the same bits."""
    dtype = getattr(torch, dtype)
    heads, kv, hd, page = 8, 2, 128, 16
    seqs = R.Seqs([n, n], [max(n, 400), n + 310], page, seed=12)
    cache, kk, vv = filled(seqs, kv, hd, 3)
    q = randn(gen(2), seqs.rows, heads, hd, dtype=dtype)
    lens = seqs.seq_lens.clone()
    table = seqs.table.clone()
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, lens, table, heads, kv, hd,
                                          out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, lens, table, heads, kv, hd,
                                          out=out)
    for cut in (0, 150):
        lens.copy_(torch.clamp(seqs.seq_lens - cut, min=n))
        want = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, seqs.offsets, lens, table, heads, kv,
                                                 hd)
        for _ in range(2):
            out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_two_streams_at_once(cuda):
    """Calls that overlap keep their own workspaces; the stream argument is the
    stream that the call's memory belongs to."""
    heads, kv, hd = 32, 8, 128
    seqs = R.Seqs([1, 1, 1], [5000, 3000, 20], 64, seed=12)
    cache, _, _ = filled(seqs, kv, hd, 3)
    qs = [randn(gen(i), 3, heads, hd) for i in range(2)]
    want = [mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd)
            for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            got[i].append(mlb.CudaPagedAttentionDeviceInput(
                qs[i], cache, 0, *seqs.where(), heads, kv, hd, stream=streams[i].cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


def test_offsets_past_32_bits(cuda):
    """Pages that start more than 4 GiB into the pool."""
    kv, hd, page, heads = 8, 128, 64, 32
    seqs = R.Seqs([1], [300], page, seed=2)
    cache = mlb.CudaPagedKvCache(1, 70000, page, kv, hd)
    assert cache.bytes() > 1 << 32
    table = (69999 - torch.arange(seqs.table.shape[1], device="cuda")).to(torch.int32)[None]
    g = gen(8)
    k, v = randn(g, 300, kv, hd), randn(g, 300, kv, hd)
    cache.AppendDevice(0, k, v, seqs.all_offsets, seqs.seq_lens, table, rope_type=mlb.ROPE_NONE)
    kk, vv = cache.ReadDevice(0, seqs.all_offsets, seqs.seq_lens, table, 300)
    assert torch.equal(vv[:40].double().cpu(), R.quantise(v[:40]))
    for n in (1, 50):
        s = R.Seqs([n], [300], page, seed=2)
        q = randn(g, n, heads, hd)
        out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, s.offsets, s.seq_lens, table, heads,
                                                kv, hd)
        check_attention(out, q, kk, vv, s, hd, torch.float32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
@pytest.mark.parametrize("n", [1, 5, 1200])
def test_scale_of_any_sign(cuda, n, scale, dtype):
    dtype = getattr(torch, dtype)
    seqs = R.Seqs([n], [max(n, 333)], 16, seed=3)
    cache, kk, vv = filled(seqs, 2, 64, 17)
    q = randn(gen(4), n, 8, 64, dtype=dtype)
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, 2, 64, scale=scale)
    check_attention(out, q, kk, vv, seqs, 64, dtype, scale=scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_largest_values(cuda, dtype):
    """Scales up to fp16's largest, next to ordinary ones."""
    dtype = getattr(torch, dtype)
    kv, hd, length = 2, 64, 1500
    g = gen(5)
    k, v = randn(g, length, kv, hd), randn(g, length, kv, hd)
    k[100:110] *= 3e4
    v[40:50] *= 1e5
    v[200, 0, 3] = 1e9  # past the format: kept at its largest scale
    for n in (1, 70, 1300):
        seqs = R.Seqs([n], [length], 32, seed=3)
        cache = mlb.CudaPagedKvCache(1, seqs.n_pages, 32, kv, hd)
        cache.AppendDevice(0, k, v, *seqs.whole(), rope_type=mlb.ROPE_NONE)
        kk, vv = cache.ReadDevice(0, *seqs.whole(), length)
        assert torch.isfinite(vv).all() and vv.max() == 7 * 65504
        q = randn(g, n, 8, hd, dtype=dtype) * 1e-3
        out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 8, kv, hd)
        check_attention(out, q, kk, vv, seqs, hd, dtype)


def test_nothing_to_do(cuda):
    cache = mlb.CudaPagedKvCache(1, 2, 16, 2, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    none = (torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, 1, **i32))
    x = torch.empty(0, 2, 64, device="cuda")
    cache.AppendDevice(0, x, x, *none, q=x)
    assert cache.ReadDevice(0, *none, 0)[0].shape == (0, 2, 64)
    assert (cache.ReadDevice(0, *none, 3)[1] == 0).all()
    assert mlb.CudaPagedAttentionDeviceInput(x, cache, 0, *none, 2, 2, 64).shape == x.shape
    # sequences without rows, and a row of a sequence of length zero
    one = (torch.zeros(2, **i32), torch.zeros(1, **i32), torch.zeros(1, 1, **i32))
    mlb.CudaPagedAttentionDeviceInput(x, cache, 0, *one, 2, 2, 64)
    row = torch.ones(1, 2, 64, device="cuda")
    offs = torch.tensor([0, 1], **i32)
    out = mlb.CudaPagedAttentionDeviceInput(row, cache, 0, offs, one[1], one[2], 2, 2, 64)
    assert (out == 0).all()


def test_refusals(cuda):
    cache = mlb.CudaPagedKvCache(1, 4, 16, 2, 64)
    seqs = R.Seqs([2], [20], 16)
    k = torch.zeros(2, 2, 64, device="cuda")
    q = torch.zeros(2, 4, 64, device="cuda")
    at = seqs.where()

    def refused(text, f, kind=mlb.MlbError):
        with pytest.raises(kind, match=text):
            f()

    A = mlb.CudaPagedAttentionDeviceInput
    refused("layer out of range", lambda: cache.AppendDevice(1, k, k, *at), mlb.MlbRangeError)
    refused("expected k and v", lambda: cache.AppendDevice(0, q, q, *at))
    refused("expected float32 or bfloat16", lambda: cache.AppendDevice(0, k.half(), k.half(), *at))
    refused("differ in type", lambda: cache.AppendDevice(0, k, k.bfloat16(), *at))
    refused("expected q", lambda: cache.AppendDevice(0, k, k, *at, q=q.bfloat16()))
    refused("q_out without q", lambda: cache.AppendDevice(0, k, k, *at, q_out=q))
    refused("q_out must be", lambda: cache.AppendDevice(0, k, k, *at, q=q, q_out=q[:1]))
    refused("unknown rope type", lambda: cache.AppendDevice(0, k, k, *at, rope_type=7))
    refused("theta must be", lambda: cache.AppendDevice(0, k, k, *at, theta=0.0))
    refused("is on cpu", lambda: cache.AppendDevice(0, k.cpu(), k.cpu(), *at))
    refused("is on cpu", lambda: cache.AppendDevice(0, k, k, *at, q=q.cpu()))
    refused("int32 seq_lens", lambda: cache.AppendDevice(0, k, k, at[0], at[1].long(), at[2]))
    refused("int32 row_offsets", lambda: cache.AppendDevice(0, k, k, at[0][:1], at[1], at[2]))
    refused("int32 page_table", lambda: A(q, cache, 0, at[0], at[1],
                                          at[2].repeat(2, 1), 4, 2, 64))
    refused("divisible", lambda: A(q[:, :3], cache, 0, *at, 3, 2, 64))
    refused("does not match attention shape", lambda: A(q, cache, 0, *at, 4, 1, 64))
    refused("expected q", lambda: A(q, cache, 0, *at, 2, 2, 64))
    refused("out must be", lambda: A(q, cache, 0, *at, 4, 2, 64, out=q.bfloat16()))
    refused("must not overlap", lambda: A(q, cache, 0, *at, 4, 2, 64, out=q))
    refused("scale must be finite", lambda: A(q, cache, 0, *at, 4, 2, 64, scale=math.inf))
    refused("cache is empty", lambda: A(q, mlb.CudaPagedKvCache(), 0, *at, 4, 2, 64))
    refused("multiple of 16", lambda: mlb.CudaPagedKvCache(1, 4, 24, 2, 64))
    refused("head_dim must be", lambda: mlb.CudaPagedKvCache(1, 4, 16, 2, 136))


def test_serving_run(cuda):
    """A prompt, then tokens one by one: append, attention over the layers of a
    small stack, then log probabilities, against 64-bit attention over what the
    cache holds; drafted tokens checked together give the same rows."""
    heads, kv, hd, page, layers, vocab = 8, 2, 64, 16, 2, 999
    steps = [[20, 1], [1, 1], [1, 1], [4, 3]]
    g = gen(40)
    ids = torch.randperm(16, device="cuda", generator=g).to(torch.int32).view(2, 8)
    cache = mlb.CudaPagedKvCache(layers, 16, page, kv, hd)
    proj = randn(g, heads * hd, vocab) * 0.1
    lens = [0, 0]
    keep = [([], []) for _ in range(layers)]
    for new in steps:
        lens = [a + b for a, b in zip(lens, new)]
        i32 = dict(dtype=torch.int32, device="cuda")
        offs = torch.tensor([0, new[0], sum(new)], **i32)
        where = (offs, torch.tensor(lens, **i32), ids)
        x = randn(g, sum(new), heads, hd)
        for layer in range(layers):
            k, v = randn(g, sum(new), kv, hd), randn(g, sum(new), kv, hd)
            q = cache.AppendDevice(layer, k, v, *where, q=x)
            x = mlb.CudaPagedAttentionDeviceInput(q, cache, layer, *where, heads, kv, hd)
            row = 0
            for s in range(2):
                whole = torch.tensor([0, lens[s]], **i32)
                kk, vv = cache.ReadDevice(layer, whole, where[1][s:s + 1], ids[s:s + 1], lens[s])
                want, vabs, top = R.attention(q[row:row + new[s]], kk, vv, lens[s], new[s],
                                              1 / math.sqrt(hd))
                err = (x[row:row + new[s]].double().cpu() - want).abs()
                assert (err <= R.attention_bound(want, vabs, top, lens[s], torch.float32)).all()
                row += new[s]
        logits = x.flatten(1) @ proj
        tok = torch.randint(vocab, (sum(new),), device="cuda", generator=g, dtype=torch.int32)
        lp, _, top_ids, _ = mlb.CudaLogProbs(logits, tok, top_k=3)
        want = torch.log_softmax(logits.double(), -1)
        assert (lp - want.gather(1, tok.long()[:, None])[:, 0]).abs().max() < 1e-4
        assert torch.equal(top_ids[:, 0].long(), want.argmax(-1))
