"""GPU: log probabilities of given tokens, entropy, top alternatives and their gradient against the plain 64-bit forms.

Tolerances.  Forward: terms e^(x - m) carry 2^-21 relative (exponential 2^-22, its fp32 argument |x - m| 2^-24 <= 2^-19 for those
that are e^-32 or less of the sum), sums of n positive terms in per-thread partial sums of at most n / 32 and a tree add less
than 2^-24 sqrt-like growth, bounded here by 2^-18 in all; log s is then off by 2^-18 absolute, x and lse round to fp32 (2^-24
relative of magnitudes up to |lse| + 2^5).  So |error| <= 2^-17 + 2^-22 |value| for lse and log probabilities; the entropy is
a sum of p |log p| whose terms carry the same relative error: 2^-17 (1 + entropy).
Gradient: p has relative error 2^-21 + |log p| 2^-23, and the factor |u| + |w| (|log p| + H) the rounding of its sum; the output
rounds once: |error| <= eps |d| + p (|u| + |w| (|log p| + H)) (2^-19 + |log p| 2^-22) + 2^-24 |u|, plus half the type's smallest subnormal."""
import numpy as np
import pytest

import kv_oracle
from pyc_b200 import abi

pytestmark = pytest.mark.gpu
F32, BF16, F16 = abi.DTYPE_F32, abi.DTYPE_BF16, abi.DTYPE_F16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


def _tt(dtype):
    import torch
    return {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}[dtype]


def _logits(dtype, x, stride=None, shift=0):
    """x rounded to the type on the device, rows `stride` apart, the first value `shift` elements behind an aligned address."""
    import torch
    rows, vocab = x.shape
    stride = stride or vocab
    buf = torch.full((rows * stride + shift + 8,), 55.0, dtype=_tt(dtype), device="cuda")
    view = buf[shift:shift + rows * stride].view(rows, stride)
    view[:, :vocab] = torch.from_numpy(np.ascontiguousarray(x)).cuda().to(_tt(dtype))
    return buf, view, view[:, :vocab].double().cpu().numpy()


def _score(backend, dtype, x, tokens, k, stride=None, shift=0, optional=True):
    import torch
    buf, view, vals = _logits(dtype, x, stride, shift)
    rows, vocab = x.shape
    t = torch.tensor(np.asarray(tokens), dtype=torch.int32, device="cuda")
    lp, ent, lse = (torch.full((rows + 1,), 7.0, device="cuda") for _ in range(3))
    ids, top = torch.full((rows, k), 7, dtype=torch.int32, device="cuda"), torch.full((rows, k), 7.0, device="cuda")
    backend.token_logprobs(dtype, rows, vocab, view.data_ptr(), t.data_ptr(), lp.data_ptr(), entropy=ent.data_ptr() if optional else None,
                           lse=lse.data_ptr() if optional else None, top_k=k, top_ids=ids.data_ptr() if k else None,
                           top_logprobs=top.data_ptr() if k else None, row_stride=view.stride(0) if rows > 1 else vocab,
                           stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert lp[rows] == ent[rows] == lse[rows] == 7.0
    return vals, [v.double().cpu().numpy() for v in (lp[:rows], ent[:rows], lse[:rows])] + [ids.cpu().numpy(), top.double().cpu().numpy()]


def _close(got, want, tol):
    special = ~np.isfinite(want)
    assert np.array_equal(got[special], want[special], equal_nan=True)
    err = np.abs(got[~special] - want[~special])
    assert (err <= np.broadcast_to(tol, want.shape)[~special]).all(), f"off by {err.max()}"


def _check(vals, got, tokens, k, optional=True):
    want = kv_oracle.scores(vals, tokens, k)
    for i in (0, 2) if optional else (0,):
        _close(got[i], want[i], 2.0 ** -17 + 2.0 ** -22 * np.abs(np.nan_to_num(want[i], posinf=0, neginf=0)))
    if optional:
        _close(got[1], want[1], 2.0 ** -17 * (1 + np.abs(want[1])))
    else:
        assert (got[1] == 7.0).all() and (got[2] == 7.0).all()
    assert np.array_equal(got[3], want[3])
    _close(got[4], want[4], 2.0 ** -17 + 2.0 ** -22 * np.abs(np.nan_to_num(want[4], posinf=0, neginf=0)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, vocab, k", [(1, 1, 1), (1, 1, 0), (3, 7, 7), (5, 33, 32), (2, 1000, 0), (17, 4096, 20), (1, 50001, 5), (3, 70003, 32), (1, 131072, 20),
                                            (300, 511, 8), (2, 262147, 10)])
def test_scores(backend, dtype, rows, vocab, k):
    rng = np.random.default_rng(vocab + rows)
    x, tokens = 4 * rng.standard_normal((rows, vocab)), rng.integers(0, vocab, rows)
    vals, got = _score(backend, dtype, x, tokens, k)
    _check(vals, got, tokens, k)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shift, extra", [(1, 0), (0, 3), (5, 7), (0, 24)])
def test_scores_of_unaligned_and_strided_rows(backend, dtype, shift, extra):
    rng = np.random.default_rng(shift)
    x, tokens = 3 * rng.standard_normal((6, 2999)), rng.integers(0, 2999, 6)
    vals, got = _score(backend, dtype, x, tokens, 9, stride=2999 + extra, shift=shift)
    _check(vals, got, tokens, 9)
    vals, got = _score(backend, dtype, x, tokens, 9, stride=2999 + extra, shift=shift, optional=False)
    _check(vals, got, tokens, 9, optional=False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_ties_go_to_the_lower_index(backend, dtype):
    rng = np.random.default_rng(2)
    x = rng.integers(-3, 4, (12, 9000)).astype(np.float64)             # thousands of equal logits
    x[1] = 0.0
    x[2, ::2] = -0.0                                                   # minus zero equals zero
    x[2, 1::2] = 0.0
    x[3] = np.arange(9000) // 100 / 8                                  # ascending: each new one is among the best so far
    x[4] = -np.arange(9000) / 64
    x[5] = -np.inf
    x[5, 8000:8007] = 1.0
    tokens = rng.integers(0, 9000, 12)
    vals, got = _score(backend, dtype, x, tokens, 32)
    _check(vals, got, tokens, 32)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [40, 5000, 140001])
def test_masked_and_broken_rows(backend, dtype, vocab):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((12, vocab))
    low = {F32: -3.4028234663852886e38, BF16: -3.3895313892515355e38, F16: -65504.0}[dtype]
    x[0] = -np.inf                                                     # nothing is left
    x[1, :] = -np.inf
    x[1, vocab // 2] = 2.0                                             # one token is left: entropy 0
    x[2, 3] = np.nan
    x[3, vocab - 1] = np.inf
    x[4, : vocab // 2] = -np.inf                                       # the first half is masked
    x[5, vocab // 3:] = -np.inf
    x[6] = low                                                         # masked by the type's lowest value, all of it: uniform
    x[7, ::2] = low
    x[8] = -low                                                        # the largest value
    x[9] = -np.inf
    x[9, -1] = -np.inf
    x[10, 1] = np.nan
    x[10, 0] = np.inf
    tokens = rng.integers(0, vocab, 12)
    tokens[4], tokens[9], tokens[11], tokens[5] = 0, -1, vocab, -5     # a masked token, and no token
    vals, got = _score(backend, dtype, x, tokens, 5)
    _check(vals, got, tokens, 5)
    assert got[1][0] == 0.0 and got[1][1] == 0.0 and got[0][9] == 0.0 and got[0][11] == 0.0


def test_sharp_and_flat_distributions(backend):
    x = np.zeros((4, 20000))
    x[1, 77] = 80.0
    x[2] = np.linspace(-60, 60, 20000)
    x[3] = 1e4 + np.linspace(0, 1, 20000)
    vals, got = _score(backend, F32, x, [5, 77, 19999, 3], 3)
    _check(vals, got, [5, 77, 19999, 3], 3)


def _gradient(backend, dtype, x, tokens, u, w, stride=None, shift=0, in_place=False, no_u=False, no_w=False):
    import torch
    buf, view, vals = _logits(dtype, x, stride, shift)
    rows, vocab = x.shape
    lp, ent, lse, _, _ = kv_oracle.scores(vals, tokens, 1)
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.float32, device="cuda")
    t, z, h, du, dw = torch.tensor(np.asarray(tokens), dtype=torch.int32, device="cuda"), dev(lse), dev(ent), dev(u), dev(w)
    dbuf, out, _ = (buf, view, None) if in_place else _logits(dtype, np.full(x.shape, 9.0), stride, shift)
    s = view.stride(0) if rows > 1 else vocab
    backend.token_logprobs_backward(dtype, rows, vocab, view.data_ptr(), t.data_ptr(), z.data_ptr(), None if no_w else h.data_ptr(),
                                    None if no_u else du.data_ptr(), None if no_w else dw.data_ptr(), out.data_ptr(), row_stride=s, grad_stride=s,
                                    stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (out[:, vocab:] == 55.0).all() and (dbuf[shift + rows * out.shape[1]:] == 55.0).all() and (dbuf[:shift] == 55.0).all()
    z64, h64 = z.double().cpu().numpy(), h.double().cpu().numpy()
    u64, w64 = (np.zeros(rows) if no_u else du.double().cpu().numpy()), (np.zeros(rows) if no_w else dw.double().cpu().numpy())
    return out[:, :vocab].double().cpu().numpy(), vals, z64, h64, u64, w64


def _check_gradient(dtype, got, vals, tokens, z, h, u, w):
    want = kv_oracle.score_gradient(vals, tokens, z, h, u, w)
    with np.errstate(invalid="ignore"):
        l = np.where(np.isfinite(vals - z[:, None]), vals - z[:, None], 0.0)
    p = np.exp(l) * np.isfinite(vals) * np.isfinite(z)[:, None]
    factor = np.abs(u)[:, None] + np.abs(w)[:, None] * (np.abs(l) + np.abs(h)[:, None])
    tol = HALF_STEP[dtype] * np.abs(want) + p * factor * (2.0 ** -19 + np.abs(l) * 2.0 ** -22) + 2.0 ** -24 * np.abs(u)[:, None] + TINY[dtype]
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    off = np.where(nan, 0, np.abs(got - want) / tol)
    assert off.max() <= 1.0, f"error is {off.max():.2f} of the tolerance"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, vocab, stride, shift", [(1, 1, None, 0), (3, 7, None, 0), (5, 1000, None, 0), (4, 4099, None, 0), (6, 2999, 3005, 3), (2, 70003, 70008, 0), (300, 64, None, 0),
                                                        (1, 131072, None, 0)])
def test_gradient(backend, dtype, rows, vocab, stride, shift):
    rng = np.random.default_rng(rows + vocab)
    x, tokens = 3 * rng.standard_normal((rows, vocab)), rng.integers(0, vocab, rows)
    u, w = rng.standard_normal(rows), rng.standard_normal(rows)
    got, *rest = _gradient(backend, dtype, x, tokens, u, w, stride, shift)
    _check_gradient(dtype, got, rest[0], tokens, *rest[1:])
    same, *_ = _gradient(backend, dtype, x, tokens, u, w, stride, shift, in_place=True)
    assert np.array_equal(got, same)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gradient_of_masked_rows_and_missing_tokens(backend, dtype):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 3001))
    x[0] = -np.inf
    x[1, ::2] = -np.inf
    x[2] = -np.inf
    x[2, 9] = 1.0
    tokens = np.array([4, 2, 9, -1, 3001, 0])
    u, w = rng.standard_normal(6), rng.standard_normal(6)
    for skip in (dict(), dict(no_u=True), dict(no_w=True)):
        got, *rest = _gradient(backend, dtype, x, tokens, u, w, **skip)
        _check_gradient(dtype, got, rest[0], tokens, *rest[1:])
    assert (got[0] == 0).all()


def test_gradient_against_differences(backend):
    """d(loss)/dx from central differences of the forward call itself, on logits that differences of fp32 results can resolve."""
    rng = np.random.default_rng(6)
    rows, vocab, step = 3, 23, 2.0 ** -5
    x, tokens, u, w = rng.standard_normal((rows, vocab)), np.array([0, 7, 22]), np.array([1.0, -0.7, 0.3]), np.array([0.5, 1.0, -2.0])
    got, vals, *_ = _gradient(backend, F32, x, tokens, u, w)
    def loss(y):
        _, (lp, ent, *_r) = _score(backend, F32, y, tokens, 0)
        return u * lp + w * ent
    for j in range(vocab):
        e = np.zeros((rows, vocab))
        e[:, j] = step
        slope = (loss(vals + e) - loss(vals - e)) / (2 * step)
        # third derivatives of both terms are below 8 in size: step^2 / 6 * 8 * 3; results are good to 2^-16, over 2 * step
        assert np.abs(slope - got[:, j]).max() <= step ** 2 / 6 * 8 * 3 + 2 * 3 * 2.0 ** -16 / (2 * step)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, vocab", [(3, 60000), (400, 9000)])
def test_top_of_rows_masked_down_to_a_few_tokens(backend, dtype, rows, vocab):
    """Fewer unmasked tokens than alternatives asked for: the masked ones follow by index, the lowest value before -inf."""
    rng = np.random.default_rng(8)
    low = {F32: -3.4028234663852886e38, BF16: -3.3895313892515355e38, F16: -65504.0}[dtype]
    x = np.full((rows, vocab), -np.inf)
    for r in range(rows):
        x[r, rng.choice(vocab, r % 25, replace=False)] = rng.standard_normal(r % 25)
        if r % 3 == 1:
            x[r, rng.choice(vocab, 5, replace=False)] = low
        if r % 3 == 2:
            x[r, x[r] == -np.inf] = low
    tokens = rng.integers(0, vocab, rows)
    vals, got = _score(backend, dtype, x, tokens, 20)
    _check(vals, got, tokens, 20)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [2048 * 9, 2048 * 40 + 5])
def test_top_of_rows_whose_large_logits_lie_in_few_threads_shares(backend, dtype, vocab):
    """Larger logits at the same places of every 2048: more of them than candidates are kept for; and a rising run."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((300, vocab))
    x[0, np.arange(vocab) % 2048 < 200] += 20.0
    x[1, np.arange(vocab) % 1024 < 60] += 20.0
    x[2, np.arange(vocab) % 2048 < 8] = 9.0
    x[3] = np.arange(vocab) / 4096
    x[4, 5000:9000] = 30 + np.arange(4000) / 500
    x[5] = np.where(np.arange(vocab) % 3 == 0, 5.0, -5.0)
    tokens = rng.integers(0, vocab, 300)
    vals, got = _score(backend, dtype, x[:8], tokens[:8], 32)            # a cluster per row
    _check(vals, got, tokens[:8], 32)
    vals, got = _score(backend, dtype, x, tokens, 32)                    # a CTA per row
    _check(vals[:8], [g[:8] for g in got], tokens[:8], 32)
