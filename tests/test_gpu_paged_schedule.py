"""Paged attention where its division of the work turns over: more units than a CTA lists
at a time, runs longer than its page look-ups, more sequences than a block has threads,
prompts beside decoding sequences. Against 64-bit attention within paged_ref's bound."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402
from tests import paged_ref as R  # noqa: E402
from tests.test_gpu_paged import check_attention, filled, gen, randn  # noqa: E402


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    assert mlb.paged_attention_status() == (0, 0)


def attend(new, lens, heads, kv, hd, dtype, width=None, prompt=False, page=16):
    """Checks a call; its page table is at least `width` tokens wide."""
    dtype = getattr(torch, dtype)
    assert R.prompt_form(sum(new), len(new), kv, heads // kv, dtype) == prompt
    seqs = R.Seqs(new, lens, page, seed=len(new))
    if width:
        more = width // page - seqs.table.shape[1]
        seqs.table = torch.nn.functional.pad(seqs.table, (0, more), value=-1)
    cache, kk, vv = filled(seqs, kv, hd, 61)
    q = randn(gen(62), seqs.rows, heads, hd, dtype=dtype) * 2
    out = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd)
    check_attention(out, q, kk, vv, seqs, hd, dtype)
    again = mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), heads, kv, hd)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", [128, 1024])
@pytest.mark.parametrize("heads", [32, 96])
def test_more_units_than_a_cta_lists(cuda, heads, width, dtype):
    """22400 units for at most 592 CTAs, 32 listed at a time; whole (short tables) and
    in runs that may cut them."""
    lens = [1 + (i * 29) % 77 for i in range(700)]
    attend([1] * 700, lens, heads, 32, 8, dtype, width)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [1, 3])
def test_runs_longer_than_a_look_up(cuda, new, dtype):
    """More than 32 chunks of one unit with one CTA: 256 units of 128 chunks."""
    attend([new] * 8, [8192 - 100 * i for i in range(8)], 64, 32, 8, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_run_per_head_and_many_chunks(cuda, dtype):
    """Runs that begin and end inside units of 400 chunks and more."""
    attend([1, 0, 2, 1], [40000, 3, 25617, 31999], 32, 32, 32, dtype, page=64)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (8, 4, 4)])
def test_more_sequences_than_threads(cuda, hd, heads, kv, dtype):
    """The search over more than 128 sequences, with units cut between CTAs."""
    lens = [1 + (i * i * 37) % (3000 if i % 7 == 0 else 300) for i in range(300)]
    attend([(i % 5 != 3) * (1 + i % 2) for i in range(300)], lens, heads, kv, hd, dtype, 3104)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_more_prompts_than_threads(cuda, dtype):
    """More than 416 sequences in the prompt form, some without rows."""
    new = [0 if i % 11 == 4 else 30 + i % 20 for i in range(500)]
    attend(new, [n + i % 40 for i, n in enumerate(new)], 32, 2, 32, dtype, prompt=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,lens", [
    ([512, 1], [512, 9000]), ([1, 700, 1, 3], [5000, 900, 17, 6001])])
def test_prompts_beside_decoding_sequences(cuda, new, lens, dtype):
    attend(new, lens, 32, 8, 128, dtype, prompt=True, page=64)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [32, 128])
def test_prompts_on_two_streams(cuda, hd, dtype):
    """Calls that overlap share the SMs' tensor memory, which one CTA takes whole."""
    dtype = getattr(torch, dtype)
    seqs = R.Seqs([400, 300, 350], [400, 700, 360], 32, seed=3)
    cache, _, _ = filled(seqs, 4, hd, 63)
    qs = [randn(gen(i), seqs.rows, 16, hd, dtype=dtype) for i in range(2)]
    assert R.prompt_form(seqs.rows, 3, 4, 4, dtype)
    want = [mlb.CudaPagedAttentionDeviceInput(q, cache, 0, *seqs.where(), 16, 4, hd) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            got[i].append(mlb.CudaPagedAttentionDeviceInput(
                qs[i], cache, 0, *seqs.where(), 16, 4, hd, stream=streams[i].cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
