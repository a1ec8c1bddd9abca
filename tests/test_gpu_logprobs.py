"""Log probabilities, entropy and alternatives against 64-bit forms.

The error bound: x - m is off by up to |x| 2^-24, y by |y| 2^-24 more,
exponentials are off by 2^-22, a thread adds vocab / 512 of them (vocab / 512
2^-24), and the sums join in 16 steps.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import mini_llama_b200 as mlb  # noqa: E402


def want_rows(x, tokens, k):
    x = x.double()
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = x - lse
    p = lp.exp()
    ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return (lp.gather(1, tokens.long()[:, None])[:, 0], ent, ids[:, :k].int(),
            (top - lse)[:, :k], p, lp)


def check(x, tokens, k):
    got = mlb.CudaLogProbs(x, tokens, top_k=k)
    chosen, ent, ids, top, p, lp = want_rows(x, tokens, k)
    big = x.double().masked_fill(~torch.isfinite(x), 0).abs().amax(-1)
    n = x.shape[1] / 512 + 32
    tol = (4 * big + n) * 2.0 ** -23
    dead = torch.isinf(chosen)
    assert torch.equal(got[0].double()[dead], chosen[dead])
    err = (got[0].double() - chosen).abs()[~dead]
    assert (err <= tol[~dead] + chosen[~dead].abs() * 2.0 ** -22).all(), err.max()
    spread = (p * torch.where(p > 0, lp.abs(), torch.zeros_like(lp))).sum(-1)
    assert ((got[1].double() - ent).abs() <= tol + n * (spread + 2) * 2.0 ** -22).all()
    assert torch.equal(got[2], ids)
    if k:
        fin = torch.isfinite(top)
        t = (got[3].double() - top).abs()
        assert (t <= tol[:, None] + top.abs() * 2.0 ** -22)[fin].all()
        assert torch.equal(got[3].double()[~fin], top[~fin])
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,k", [
    (1, 1, 1), (3, 7, 3), (2, 33, 32), (5, 511, 32), (1, 4099, 20), (1, 16384, 5), (1, 32771, 32),
    (2, 128256, 20), (33, 152064, 5), (150, 9001, 2), (600, 1000, 1), (64, 5000, 0), (7, 2048, 31)])
def test_logprobs(cuda, rows, vocab, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(getattr(torch, dtype))
    tok = torch.randint(vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    a = check(x, tok, k)
    b = mlb.CudaLogProbs(x, tok, top_k=k)
    for u, v in zip(a, b):
        assert torch.equal(u, v)


@pytest.mark.parametrize("vocab", [5000, 40000, 128256])
@pytest.mark.parametrize("kind", ["equal", "periodic", "ascending", "descending", "two",
                                  "huge", "zeros"])
def test_orders_and_ties(cuda, kind, vocab):
    """Logits that defeat a guess of the k-th largest; ties go to the lower index."""
    i = torch.arange(vocab, device="cuda")
    x = {"equal": torch.full((vocab,), -3.25, device="cuda"),
         "periodic": ((i * 7919) % 2048).float() / 512,
         "ascending": i.float() / vocab * 30, "descending": -i.float() / vocab * 30,
         "two": (i % 3 == 1).float() * 5, "huge": (i % 97).float() * 1e30,
         "zeros": torch.where(i % 2 == 0, 0.0, -0.0)}[kind]
    x = torch.stack([x, x.flip(0)])
    tok = torch.tensor([0, vocab - 1], dtype=torch.int32, device="cuda")
    if kind == "huge":  # the largest logits alone count
        got = mlb.CudaLogProbs(x, tok, top_k=20)
        assert torch.equal(got[2], torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :20].int())
        n = (x[0] == x[0].max()).sum().double()
        assert (got[1].double() - n.log()).abs().max() < 1e-5
        return
    check(x, tok, 20)
    check(x.repeat(200, 1), tok.repeat(200), 32)


def test_masked_logits(cuda):
    """-inf has probability zero; type-lowest values underflow to it."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(4, 5000, device="cuda", generator=g).to(dtype)
        x[0, 100:] = -math.inf
        x[1, :4990] = -math.inf
        x[2, 7:] = torch.finfo(dtype).min
        x[3, 1:] = -math.inf
        tok = torch.tensor([5, 4995, 3, 0], dtype=torch.int32, device="cuda")
        got = check(x, tok, 10)
        assert got[0][3] == 0 and got[1][3] == 0
    assert torch.equal(mlb.CudaLogProbs(x, torch.full_like(tok, 200))[0][0], torch.tensor(
        -math.inf, device="cuda"))


@pytest.mark.parametrize("vocab", [300, 40000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_extreme_logits_next_to_masked_ones(cuda, dtype, vocab):
    dtype = getattr(torch, dtype)
    x = torch.full((3, vocab), -math.inf, device="cuda", dtype=dtype)
    x[0, :8], x[1, 5:7] = 2e38, 3e38
    x[1, ::2], x[2, 1::3] = torch.finfo(dtype).min, torch.finfo(dtype).min
    tok = torch.tensor([3, 5, 1], dtype=torch.int32, device="cuda")
    lp, ent, ids, _ = mlb.CudaLogProbs(x, tok, top_k=4)
    # 8 equal logits; one or two of 3e38 (index 6 is even: the lowest); every third
    want = [math.log(8), 0.0, math.log(len(range(1, vocab, 3)))]
    for r in range(3):
        assert abs(lp[r] + want[r]) < 1e-5 and abs(ent[r] - want[r]) < 1e-5
    assert ids.tolist() == [[0, 1, 2, 3], [5, 0, 2, 4], [1, 4, 7, 10]]


def test_rows_without_a_number(cuda):
    x = torch.zeros(4, 3000, device="cuda")
    x[0] = -math.inf
    x[1, 5] = math.nan
    x[2, 9] = math.inf
    tok = torch.tensor([0, 1, 9, 3], dtype=torch.int32, device="cuda")
    lp, ent, ids, top = mlb.CudaLogProbs(x, tok, top_k=3)
    assert torch.isnan(lp[:3]).all() and torch.isnan(ent[:3]).all()
    assert ((ids >= -1) & (ids < 3000)).all()
    assert ids[2, 0] == 9
    assert abs(lp[3] + math.log(3000)) < 1e-5
    x = torch.full((1, 40), math.nan, device="cuda")
    x[0, 3], x[0, 30] = 1.0, 2.0
    _, _, ids, top = mlb.CudaLogProbs(x, tok[:1], top_k=4)
    assert ids.tolist() == [[30, 3, -1, -1]] and torch.isnan(top).all()


def test_padded_rows(cuda):
    x = torch.randn(3, 100, device="cuda")
    tok = torch.tensor([-1, 100, 5], dtype=torch.int32, device="cuda")
    lp, ent, _, _ = mlb.CudaLogProbs(x, tok)
    assert torch.isnan(lp[:2]).all() and torch.isfinite(lp[2]) and torch.isfinite(ent).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_alignment(cuda, dtype):
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(7)
    base = torch.randn(6, 4111, device="cuda", generator=g).to(dtype)
    tok = torch.randint(4000, (6,), device="cuda", generator=g, dtype=torch.int32)
    for off in range(9):
        check(base[:, off:off + 4001], tok, 7)
    check(base.t().contiguous().t()[:, :4001], tok, 7)
    check(base[::2, :4001], tok[::2].contiguous(), 7)
    check(base[:1].expand(6, 4111), tok, 7)
    one = mlb.CudaLogProbs(base[2], tok[2:3], top_k=2)
    all_ = mlb.CudaLogProbs(base, tok, top_k=2)
    for a, b in zip(one, all_):
        assert torch.equal(a[0], b[2])


def test_graph_and_stream(cuda):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(2, 70000, device="cuda", generator=g)
    tok = torch.tensor([3, 5], dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = mlb.CudaLogProbs(x, tok, top_k=4, stream=s.cuda_stream)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = mlb.CudaLogProbs(x, tok, top_k=4)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, cap):
        assert torch.equal(a, b)
    x.mul_(2)
    graph.replay()
    want = mlb.CudaLogProbs(x, tok, top_k=4)
    torch.cuda.synchronize()
    for a, b in zip(want, cap):
        assert torch.equal(a, b)


def test_no_rows_and_refusals(cuda):
    x = torch.zeros(2, 50, device="cuda")
    tok = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert mlb.CudaLogProbs(x[:0], tok[:0], top_k=3)[2].shape == (0, 3)
    for text, call in (("top_k must be", lambda: mlb.CudaLogProbs(x, tok, top_k=33)),
                       ("top_k must be", lambda: mlb.CudaLogProbs(x[:, :4], tok, top_k=5)),
                       ("expected float32", lambda: mlb.CudaLogProbs(x.half(), tok)),
                       ("int32 tokens", lambda: mlb.CudaLogProbs(x, tok.long())),
                       ("int32 tokens", lambda: mlb.CudaLogProbs(x, tok[:1])),
                       ("is on cpu", lambda: mlb.CudaLogProbs(x, tok.cpu())),
                       ("expected logits", lambda: mlb.CudaLogProbs(x[:, :0], tok)),
                       ("must be on a CUDA device", lambda: mlb.CudaLogProbs(x.cpu(), tok.cpu()))):
        with pytest.raises(mlb.MlbError, match=text):
            call()
