"""Log-probabilities, entropy, rank and alternatives of logits against 64-bit restatements: ties, forbidden tokens, NaN and
infinities, odd vocabularies, strides and alignments."""
import numpy as np
import pytest
import torch

from ferrum_gpu_b200 import CudaError, LogProbs, _ffi, logprobs

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _check(dev, logits, targets, top, vocab=None):
    """`logits`: a device tensor of rows; every output against the definitions in numpy's float64."""
    rows = logits.shape[0]
    n = logits.shape[1] if vocab is None else vocab
    out = LogProbs.new(dev, rows, top)
    t = torch.tensor(targets, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    logprobs(dev, logits, t, out, vocab=vocab)
    dev.sync()
    x = logits[:, :n].float().cpu().numpy().astype(np.float64)
    lp, en, rank, ti, tl = (a.cpu().numpy() for a in (out.logprob, out.entropy, out.rank, out.top_index, out.top_logprob))
    with np.errstate(all="ignore"):
        for r in range(rows):
            row = x[r]
            order = sorted((i for i in range(n) if not np.isnan(row[i])), key=lambda i: (-row[i], i)) if n <= 4096 else \
                np.lexsort((np.arange(n), -row))[:n - int(np.isnan(row).sum())].tolist()
            m = row[order[0]] if order else np.nan
            base = 0.0 if m == -np.inf else m
            e = np.exp(row - base)
            s = e.sum()
            ls = 0.0 if s == 0 else np.log(s)
            want_top = (order + [-1] * top)[:top]
            assert ti[r].tolist() == want_top, r
            # f32: the difference of two logits rounded once, a sum of positive terms that a thread adds at most 512 one
            # behind the other (the exponentials themselves to 2 units), its logarithm
            def near(got, want):
                if np.isnan(want) or np.isinf(want):
                    return np.array_equal(got, want, equal_nan=True) if np.isnan(want) else got == want
                return abs(got - want) <= 2.0 ** -24 * (600 + 2 * abs(want) + abs(ls))
            for j, i in enumerate(want_top):
                assert near(tl[r, j], row[i] - base - ls if i >= 0 else -np.inf), (r, j)
            if 0 <= targets[r] < n:
                v = row[targets[r]]
                assert near(lp[r], v - base - ls), (r, lp[r], v - base - ls)
                want_rank = len(order) if np.isnan(v) else int((row > v).sum() + (row[:targets[r]] == v).sum())
                assert rank[r] == want_rank, r
            else:
                assert np.isnan(lp[r]) and rank[r] == -1
            want_h = 0.0 if s == 0 else ls - np.where(e == 0, 0.0, e * (row - base)).sum() / s
            if np.isnan(want_h):
                assert np.isnan(en[r])
            else:
                # both terms of the difference are sums as above, the second weighted by |x - m|
                spread = np.where(e == 0, 0.0, -e * (row - base)).sum() / (s or 1.0)
                assert abs(en[r] - want_h) <= 2.0 ** -24 * 600 * (1 + abs(ls) + 2 * spread), (r, en[r], want_h)


def _randn(seed, rows, n, dtype="f32", scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, n, device="cuda", generator=g) * scale).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 32000, 5), (3, 50257, 20), (2, 151936, 32), (70, 1000, 1), (5, 4097, 0), (400, 257, 3)])
def test_random_rows(dev, dtype, rows, vocab, top):
    _check(dev, _randn(vocab, rows, vocab, dtype), [(i * 7919) % vocab for i in range(rows)], top)


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 31, 32, 33, 255, 256, 1023, 1025, 2047, 8191, 8193, 16385])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_vocabularies(dev, vocab, dtype):
    _check(dev, _randn(vocab, 3, vocab, dtype), [0, vocab - 1, vocab // 2], 32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(1, 0), (8, 0), (0, 1), (3, 5), (64, 3)])
def test_strides_and_alignments(dev, dtype, pad, shift):
    rows, vocab = 5, 5001
    flat = _randn(1, 1, rows * (vocab + pad) + shift, dtype)[0]
    x = flat[shift:].view(rows, vocab + pad)
    x[:, vocab:] = float("nan")  # what lies behind a row is not read
    _check(dev, x, [0, 5000, 17, 4999, 2500], 10, vocab=vocab)
    _check(dev, x[:, :vocab], [5000, 0, 1, 2, 3], 2)


@pytest.mark.parametrize("vocab", [40, 3000, 70001])
def test_ties_go_to_the_lowest_index(dev, vocab):
    g = torch.Generator(device="cuda").manual_seed(1)
    few = torch.randint(0, 5, (4, vocab), device="cuda", generator=g).float()  # thousands of equal logits
    few[1] = 2.5
    few[2] = torch.where(torch.arange(vocab, device="cuda") % 3 == 0, 0.0, -0.0)  # -0 equals +0
    few[3] = torch.arange(vocab, device="cuda").flip(0).float()
    _check(dev, few, [vocab - 1, vocab // 2, vocab - 1, 0], 32)
    _check(dev, few.to(torch.bfloat16), [1, vocab // 2, 2, vocab - 1], 32)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [50, 2000, 40000])
def test_forbidden_tokens(dev, dtype, vocab):
    x = _randn(2, 7, vocab, dtype)
    x[0, 1:] = -float("inf")          # one token is left
    x[1] = -float("inf")              # none
    x[2, ::2] = -float("inf")
    x[3, :-3] = -float("inf")         # fewer than are listed
    x[4] = torch.finfo(DT[dtype]).min
    x[5, 7:] = torch.finfo(DT[dtype]).min
    _check(dev, x, [0, 3, 4, vocab - 1, 9, 3, 5], 20)
    _check(dev, x, [1, 0, 5, 0, 0, 30, vocab - 1], 5)


@pytest.mark.parametrize("vocab", [50, 40000])
def test_nan_and_infinities(dev, vocab):
    x = _randn(3, 6, vocab)
    x[0, 5] = float("nan")
    x[1, 7] = float("inf")
    x[2] = float("nan")
    x[3, 3:] = float("nan")
    x[4, ::2] = -float("inf")
    x[4, 9] = float("nan")
    x[5] *= 1e37                       # huge, finite
    _check(dev, x, [5, 7, 3, 2, 0, 9], 8)
    _check(dev, x, [6, 8, 0, 10, 9, 11], 8)


def test_certain_and_even_distributions(dev):
    x = torch.zeros(2, 100000, device="cuda")
    x[0, 777] = 200.0
    _check(dev, x, [777, 99999], 3)


def test_targets_that_are_none_and_outputs_left_out(dev):
    x = _randn(4, 4, 999)
    _check(dev, x, [-1, 999, 2 ** 31 - 1, -2 ** 31], 2)
    whole = LogProbs.new(dev, 4, 3)
    t = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    logprobs(dev, x, t, whole)
    for name in ("logprob", "entropy", "rank", "top_index", "top_logprob"):
        one = LogProbs(**{name: getattr(LogProbs.new(dev, 4, 3), name)})
        logprobs(dev, x, t, one)
        dev.sync()
        assert torch.equal(getattr(one, name), getattr(whole, name)), name
    none = LogProbs.new(dev, 4, 3)
    logprobs(dev, x, None, none)
    dev.sync()
    assert bool(none.logprob.isnan().all()) and none.rank.tolist() == [-1] * 4 and torch.equal(none.top_index, whole.top_index)


def test_rows_past_32_bits(dev):
    vocab, rows = 150001, 29000
    x = torch.zeros(rows, vocab, dtype=torch.float16, device="cuda")  # 4.35 G elements
    x[-1, 150000], x[-1, 3], x[-2, 5] = 9.0, 8.0, 7.0
    out = LogProbs.new(dev, rows, 2)
    t = torch.full((rows,), 3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    logprobs(dev, x, t, out)
    dev.sync()
    assert out.top_index[-2:].tolist() == [[5, 0], [150000, 3]] and out.rank[-2:].tolist() == [3 + 1, 1]
    assert abs(float(out.logprob[-1]) - (8 - np.log(np.exp(9) + np.exp(8) + vocab - 2))) < 1e-4
    del x
    torch.cuda.empty_cache()


def test_the_same_bits_every_time(dev):
    x = _randn(5, 9, 70001)
    outs = [LogProbs.new(dev, 9, 6) for _ in range(8)]
    t = torch.arange(9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for out in outs:
        logprobs(dev, x, t, out)
    dev.sync()
    for out in outs:
        for name in ("logprob", "entropy", "rank", "top_index", "top_logprob"):
            assert torch.equal(getattr(out, name), getattr(outs[0], name))


def test_refusals(dev):
    x = _randn(6, 2, 64)
    out = LogProbs.new(dev, 2, 3)

    def refused(code, match, *a, **kw):
        with pytest.raises(CudaError, match=match) as e:
            logprobs(dev, *a, **kw)
        assert e.value.code == code

    refused(_ffi.FC_ERR_SHAPE, "65 logits of rows of 64", x, None, out, vocab=65)
    refused(_ffi.FC_ERR_SHAPE, "0 logits", x, None, out, vocab=0)
    refused(_ffi.FC_ERR_UNSUPPORTED, "at most 32", x, None, LogProbs.new(dev, 2, 33))
    refused(_ffi.FC_ERR_UNSUPPORTED, "float32", x.double(), None, out)
    refused(_ffi.FC_ERR_SHAPE, "has 1 entries, needs 2", x, torch.zeros(1, dtype=torch.int32, device="cuda"), out)
    refused(_ffi.FC_ERR_SHAPE, "logprob has 1 entries, needs 2", x, None, LogProbs.new(dev, 1, 3))
    with pytest.raises(CudaError, match="one width"):
        LogProbs(top_index=out.top_index, top_logprob=LogProbs.new(dev, 2, 4).top_logprob)
    refused(_ffi.FC_ERR_ARG, "side by side", x.T, None, out)
    refused(_ffi.FC_ERR_ARG, "contiguous torch.int32", x, torch.zeros(2, dtype=torch.int64, device="cuda"), out)
    refused(_ffi.FC_ERR_SHAPE, "rows of 64 logits 3 apart", torch.as_strided(x, (2, 64), (3, 1)), None, out)
    nothing = LogProbs.new(dev, 0, 3)
    logprobs(dev, x[:0], None, nothing)
    dev.sync()
