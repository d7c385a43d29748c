"""GPU: block tables and slot maps, the quantising cache write and attention over the 8-bit paged cache, against the plain 64-bit
forms in kv_oracle.py.  Tables, slots, codes and scales have to be equal.

Tolerance of attention, for each output value: half a step of the output's type relative to the value; each probability is
rounded to f16 once (2^-11 relative, below 2^-14 of the largest 2^-25 absolute); the score's fp32 products and exponential add
less than 2^-18 relative (|score| stays under 2^6 here).  So |error| <= eps/2 |o| + (2^-11 + 2^-18) sum p|v| + n 2^-25 448 max vs.
The last term is taken as n 2^-25 times the largest |v| in the cache."""
import numpy as np
import pytest

import kv_oracle
from pyc_b200 import abi

pytestmark = pytest.mark.gpu
BF16, F16 = abi.DTYPE_BF16, abi.DTYPE_F16


def _torch():
    import torch
    return torch


def _tt(dtype):
    torch = _torch()
    return {BF16: torch.bfloat16, F16: torch.float16, abi.DTYPE_F32: torch.float32}[dtype]


def _dev(x, kind=None):
    torch = _torch()
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t.to(kind) if kind is not None else t


def _sync(backend):
    _torch().cuda.synchronize()
    assert backend.device_status() == 0


# ------------------------------------------------------------------------------------------------------------------ plan
def _run_plan(backend, context, new, bs, num_blocks, width, max_tokens, seed, free=None, count=None, table=None, apart=False):
    torch = _torch()
    rng = np.random.default_rng(seed)
    R = len(context)
    order = rng.permutation(num_blocks)
    if table is None:
        table, at = np.full((R, width), -1, np.int32), 0
        for r, c in enumerate(context):
            n = -(-max(c, 0) // bs)
            table[r, :min(n, width)] = order[at:at + min(n, width)]
            at += n
        free = np.concatenate([order[at:], np.full(min(at, num_blocks), -7)])[:num_blocks].astype(np.int32)
        count = num_blocks - at if count is None else count
    d = dict(context=_dev(np.array(context, np.int32)), new=_dev(np.array(new, np.int32)), free=_dev(free), count=_dev(np.array([count], np.int32)),
             table=_dev(table), starts=_dev(np.full(R + 2, 77, np.int32)), lens=_dev(np.full(R + 1, 77, np.int32)),
             slots=_dev(np.full(max_tokens + 1, 77, np.int64)), pos=_dev(np.full(max_tokens + 1, 77, np.int32)),
             req=_dev(np.full(max_tokens + 1, 77, np.int32)), result=_dev(np.full(4, 77, np.int32)), out=_dev(np.array([77], np.int32)))
    before = table.copy()
    call = lambda: backend.kv_plan(R, bs, width, max_tokens, num_blocks, d["context"].data_ptr(), d["new"].data_ptr(), d["free"].data_ptr(),
                                   d["count"].data_ptr(), d["table"].data_ptr(), d["starts"].data_ptr(), d["lens"].data_ptr(), d["slots"].data_ptr(),
                                   d["pos"].data_ptr(), d["req"].data_ptr(), d["result"].data_ptr(),
                                   free_count_out=d["out"].data_ptr() if apart else None, stream=torch.cuda.current_stream().cuda_stream)
    call()
    if apart:                     # the count it read is as it was: the same step again
        call()
    _sync(backend)
    got = {k: v.cpu().numpy() for k, v in d.items()}
    assert got["starts"][R + 1] == got["lens"][R] == got["slots"][max_tokens] == got["pos"][max_tokens] == got["req"][max_tokens] == 77
    want_table = before.copy()
    want = kv_oracle.plan(context, new, free, max(0, min(count, num_blocks)), want_table, bs, num_blocks, max_tokens)
    return got, want, want_table, before, count


def _check_plan(got, want, want_table, count, max_tokens, apart=False):
    R = len(got["context"])
    assert got["result"].tolist()[1:] == [int(want["query_start"][-1]), want["taken"], 0]
    assert np.array_equal(got["starts"][:R + 1], want["query_start"]) and np.array_equal(got["lens"][:R], want["seq_lens"])
    assert np.array_equal(got["table"], want_table)
    assert np.array_equal(got["slots"][:max_tokens], want["slot_map"])
    assert np.array_equal(got["pos"][:max_tokens], want["positions"]) and np.array_equal(got["req"][:max_tokens], want["token_request"])
    assert got["out" if apart else "count"][0] == want["free_count"] and (not apart or got["count"][0] == count)


@pytest.mark.parametrize("R, ctx, most, bs, max_tokens", [
    (1, 0, 1, 16, 1), (1, 5, 40, 16, 64), (1, 0, 5000, 16, 5000), (3, 17, 1, 32, 3), (7, 100, 33, 64, 300), (33, 70, 1, 128, 4097),
    (1025, 40, 2, 16, 3000), (1024, 300, 1, 16, 1024), (5000, 60, 3, 16, 20000), (16384, 20, 1, 16, 16384), (2, 0, 20000, 128, 50000)])
@pytest.mark.parametrize("apart", [False, True])
def test_plan(backend, R, ctx, most, bs, max_tokens, apart):
    rng = np.random.default_rng(R + most)
    context = rng.integers(0, ctx + 1, R).tolist()
    new = rng.integers(0, most + 1, R).tolist()
    while sum(new) > max_tokens:
        new[new.index(max(new))] //= 2
    width = max(1, max(-(-(c + n) // bs) for c, n in zip(context, new)))
    need = sum(-(-(c + n) // bs) for c, n in zip(context, new))
    got, want, table, _, count = _run_plan(backend, context, new, bs, max(1, need), width, max_tokens, 5, apart=apart)
    assert got["result"][0] == 0
    _check_plan(got, want, table, count, max_tokens, apart)


@pytest.mark.parametrize("context, new, change, code", [
    ([5, -1], [1, 1], {}, 1), ([5, 2], [1, -3], {}, 1), ([60, 3], [5, 1], {}, 2), ([2**31 - 1, 3], [2**31 - 1, 1], {}, 2),
    ([5, 3], [20, 20], {}, 4), ([16, 16], [17, 17], dict(count=3), 8), ([16, 16], [1, 1], dict(count=-9), 8), ([16, 0], [64, -2], {}, 1 | 2 | 4)])
def test_plan_that_cannot_be(backend, context, new, change, code):
    safe = [c if 0 <= c <= 64 else 0 for c in context]
    if code & 4 and not code & 3:
        got, want, _, before, count = _run_plan(backend, context, new, 16, 20, 4, 39, 3)
        assert want is None
        code = 4
    else:
        rng = np.random.default_rng(3)
        order, at, table = rng.permutation(20), 0, np.full((2, 4), -1, np.int32)
        for r, c in enumerate(safe):
            n = min(4, -(-c // 16))
            table[r, :n] = order[at:at + n]
            at += n
        free = np.concatenate([order[at:], np.full(at, -7)]).astype(np.int32)
        got, want, _, before, count = _run_plan(backend, context, new, 16, 20, 4, 64 if code != 7 else 10, 3, free, change.get("count", 20 - at), table)
    assert got["result"][0] & code and got["result"][0] & 15 == got["result"][0]
    if code == 8:
        assert got["result"].tolist() == [8, 0, 0, 1 if change["count"] == 3 else 2]
    assert got["result"][1] == got["result"][2] == 0
    R = len(context)
    assert not got["starts"][:R + 1].any() and got["lens"][:R].tolist() == list(context)
    assert (got["slots"][:-1] == -1).all() and (got["req"][:-1] == -1).all() and np.array_equal(got["table"], before) and got["count"][0] == count


def test_plan_exactly_uses_up_the_pool(backend):
    got, want, table, _, count = _run_plan(backend, [16, 16], [17, 17], 16, 20, 4, 64, 3, count=None)
    assert got["result"][0] == 0
    free = np.arange(20, dtype=np.int32)
    t = np.array([[18, -1, -1, -1], [19, -1, -1, -1]], np.int32)
    got, want, table, _, count = _run_plan(backend, [16, 16], [17, 17], 16, 20, 4, 64, 3, free, 4, t)
    assert got["result"].tolist() == [0, 34, 4, 0] and got["count"][0] == 0
    _check_plan(got, want, table, count, 64)


def test_plan_with_block_ids_outside_the_pool(backend):
    free = np.array([3, 99, 5, 6, 7, 8, 9, 9], np.int32)             # 99 is taken second from the end
    t = np.array([[0, -1], [-5, -1]], np.int32)
    got, want, table, _, count = _run_plan(backend, [16, 3], [16, 14], 16, 8, 2, 40, 3, free, 2, t)
    assert got["result"][0] == 16
    _check_plan(got, want, table, count, 40)
    # request 0: 16 tokens in block 99; request 1: positions 3 .. 15 in block -5, position 16 begins block 3
    assert (got["slots"][:29] == -1).all() and got["slots"][29] == 48 and (got["slots"][30:40] == -1).all()


@pytest.mark.parametrize("R, bs, seed", [(1, 16, 0), (6, 32, 1), (700, 16, 2), (3000, 64, 3)])
def test_release_and_plan_again(backend, R, bs, seed):
    torch = _torch()
    rng = np.random.default_rng(seed)
    context = rng.integers(0, 5 * bs, R).astype(np.int32)
    held = -(-context // bs)
    num = int(held.sum()) + 10
    order, table, at = rng.permutation(num).astype(np.int32), np.full((R, 6), -1, np.int32), 0
    for r in range(R):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    free = np.concatenate([order[at:], np.full(at, -7, np.int32)]).astype(np.int32)
    finished = (rng.random(R) < 0.5).astype(np.int32)
    d = [_dev(x) for x in (finished, context, table, free, np.array([num - at], np.int32))]
    backend.kv_release(R, bs, 6, num, *[x.data_ptr() for x in d], stream=torch.cuda.current_stream().cuda_stream)
    _sync(backend)
    fin, ctx, tab, fr, cnt = [x.cpu().numpy() for x in d]
    back = [table[r, j] for r in range(R) if finished[r] for j in range(held[r])]
    assert cnt[0] == num - at + len(back)
    assert fr[:cnt[0]].tolist() == order[at:].tolist() + back and (fr[cnt[0]:] == -7).all()
    assert np.array_equal(ctx, np.where(finished, 0, context))
    assert np.array_equal(tab, np.where(finished[:, None].astype(bool), -1, table))


# ----------------------------------------------------------------------------------------------------------------- write
def _write_case(backend, dtype, slots, H, D, bs, nb, seed, x=None, stride=None, codes=None, scale=None):
    torch = _torch()
    rng = np.random.default_rng(seed)
    T = len(slots)
    if x is None:
        x = rng.standard_normal((2, T, H, D)) * np.exp2(rng.integers(-6, 7, (2, T, H, 1)))
    stride = stride or H * D
    wide = torch.zeros((2, T, stride), dtype=_tt(dtype), device="cuda")
    wide[:, :, :H * D] = _dev(x.reshape(2, T, H * D)).to(_tt(dtype))
    vals = wide[:, :, :H * D].double().cpu().numpy().reshape(2, T, H, D)
    if codes is None:
        codes = rng.integers(0, 256, (2, nb, H, bs, D)).astype(np.uint8)
        scale = np.exp2(rng.integers(-9, 3, (2, nb, H))).astype(np.float32)
    dc, ds, sl = _dev(codes), _dev(scale), _dev(np.array(slots, np.int64))
    backend.kv_write(dtype, T, H, D, bs, nb, wide[0].data_ptr(), wide[1].data_ptr(), sl.data_ptr(), dc[0].data_ptr(), dc[1].data_ptr(),
                     ds[0].data_ptr(), ds[1].data_ptr(), k_stride=stride, v_stride=stride, stream=torch.cuda.current_stream().cuda_stream)
    _sync(backend)
    want_c, want_s = codes.copy(), scale.astype(np.float64)
    for i in range(2):
        kv_oracle.write(vals[i], slots, want_c[i], want_s[i])
    got_c, got_s = dc.cpu().numpy(), ds.cpu().numpy()
    assert np.array_equal(got_s.astype(np.float64), want_s)
    nan = np.isnan(kv_oracle.VALUES)
    same = (got_c == want_c) | (nan[got_c] & nan[want_c])            # one NaN is as good as another
    assert same.all(), f"{(~same).sum()} codes differ, first at {np.argwhere(~same)[0]}"
    return got_c, got_s


def _runs(spec, bs):
    """[(block, offset, tokens)] -> slots"""
    return [b * bs + o + i for b, o, n in spec for i in range(n)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("H, D, bs", [(1, 64, 16), (3, 128, 16), (2, 64, 32), (8, 128, 64), (2, 128, 128), (1, 64, 128)])
def test_write(backend, dtype, H, D, bs):
    one = [(0, 0, 1)]
    appended = [(5, 3, 1), (2, bs - 1, 1), (7, 0, 1), (1, 1, 1)]
    prompt = [(4, 0, bs), (3, 0, bs), (0, 0, bs - 3)]
    middle = [(6, 5, bs - 5), (1, 0, bs), (8, 0, 2), (2, 2, 7)]
    for i, spec in enumerate([one, appended, prompt, middle]):
        _write_case(backend, dtype, _runs(spec, bs), H, D, bs, 9, 10 + i)


def test_write_many_ragged_requests(backend):
    rng, spec, b = np.random.default_rng(4), [], 0
    for _ in range(60):                                               # requests of random length that start anywhere in a block
        off, left = int(rng.integers(0, 16)), int(rng.integers(1, 70))
        while left:
            n = min(left, 16 - off)
            spec.append((b, off, n))
            b, left, off = b + 1, left - n, 0
    order = rng.permutation(b)
    _write_case(backend, BF16, _runs([(int(order[i]), o, n) for i, o, n in spec], 16), 4, 128, 16, b, 3)


def test_write_skips_slots_outside_the_pool_and_reads_strided_rows(backend):
    slots = [-1, 3 * 16, 3 * 16 + 1, -1, 9 * 16, -17, 2 * 16 + 4, 2 ** 40, 4 * 16 + 5, -1]       # the pool ends at 9 * 16; each block has one run
    _write_case(backend, BF16, slots, 2, 64, 16, 9, 1, stride=2 * 64 * 3 + 8)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_write_of_zeros_infinities_nan_and_extremes(backend, dtype):
    x = np.zeros((2, 12, 2, 64))
    x[:, 1, 0, :5] = [np.inf, -np.inf, np.nan, 1.0, -0.0]
    x[:, 2] = 448.0
    x[:, 3] = 448.0 * 2.0 ** -6
    x[:, 4] = 449.0 if dtype == F16 else 450.0
    x[:, 5] = np.nan
    x[:, 6] = np.inf
    x[:, 7] = 6e-8 if dtype == F16 else 1e-38
    x[:, 8] = 65504.0 if dtype == F16 else 3e38
    x[:, 9, :, ::2] = 1e-4
    x[:, 9, :, 1::2] = 400.0
    x[:, 10] = -1.0
    x[:, 11, 1] = np.linspace(-3, 3, 64)
    _write_case(backend, dtype, [b * 16 for b in range(12)], 2, 64, 16, 12, 2, x=x)               # each begins a block
    codes, scale = np.full((2, 12, 2, 16, 64), 0x38, np.uint8), np.full((2, 12, 2), 2.0 ** -8, np.float32)
    _write_case(backend, dtype, [b * 16 + 5 for b in range(12)], 2, 64, 16, 12, 2, x=x, codes=codes, scale=scale)


def test_tokens_written_one_by_one_fill_a_block(backend):
    """A block's scale only grows; every earlier code is rounded again each time it does."""
    rng = np.random.default_rng(0)
    codes, scale = rng.integers(0, 256, (2, 2, 1, 16, 64)).astype(np.uint8), np.full((2, 2, 1), 2.0 ** 40, np.float32)
    for t in range(16):
        x = rng.standard_normal((2, 1, 1, 64)) * 2.0 ** (t / 2)
        codes, scale = _write_case(backend, BF16, [16 + t], 1, 64, 16, 2, 0, x=x, codes=codes, scale=scale)


# ------------------------------------------------------------------------------------------------------------- attention
class Batch:
    """A cache with garbage (NaN codes among it) wherever no request has a token."""

    def __init__(self, context, new, Hk, G, D, bs, dtype, seed=0, nb=None, width=None, q_stride=None, out_stride=None, tail=3, sharp=1.0):
        torch = _torch()
        rng = np.random.default_rng(seed)
        self.Hk, self.G, self.D, self.bs, self.dtype = Hk, G, D, bs, dtype
        self.lens, self.starts = np.add(context, new).astype(np.int32), np.cumsum([0] + list(new)).astype(np.int32)
        need = -(-self.lens // bs)
        self.nb = nb or int(need.sum()) + 3
        self.width = width or int(max(1, need.max()))
        self.codes = rng.integers(0, 256, (2, self.nb, Hk, bs, D)).astype(np.uint8)
        self.codes[:, :, :, ::3, 1] = 0x7f
        self.scale = np.exp2(rng.integers(-9, -5, (2, self.nb, Hk))).astype(np.float32)
        self.table = np.full((len(new), self.width), -1, np.int32)
        order, at = rng.permutation(self.nb), 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
            for j in range(n):                                        # real values where there are tokens
                m = min(bs, self.lens[r] - j * bs)
                vals = np.clip(rng.standard_normal((2, Hk, m, D)) * 96, -448, 448)
                self.codes[:, self.table[r, j], :, :m] = kv_oracle.encode(vals)
        H, rows = Hk * G, int(self.starts[-1]) + tail
        self.rows = rows
        self.qs, self.os = q_stride or H * D, out_stride or H * D
        self.q = torch.zeros((rows, self.qs), dtype=_tt(dtype), device="cuda")
        self.q[:, :H * D] = _dev(rng.standard_normal((rows, H * D)) * sharp).to(_tt(dtype))
        self.scale_qk = D ** -0.5

    def run(self, backend, causal=True, max_query=None, workspace=None, lse=True):
        torch = _torch()
        H, R = self.Hk * self.G, len(self.lens)
        mq = max_query or max(1, int(np.diff(self.starts).max()))
        if workspace is None:
            workspace = torch.zeros(backend.paged_attention_workspace_bytes(R, mq, H, self.Hk, self.D), dtype=torch.uint8, device="cuda")
        self.d = [_dev(x) for x in (self.codes, self.scale, self.table, self.starts, self.lens)]
        c, s, t, st, ln = self.d
        out = torch.full((self.rows, self.os), 7.0, dtype=_tt(self.dtype), device="cuda")
        z = torch.full((self.rows, H), 7.0, device="cuda")
        backend.paged_attention(self.dtype, R, mq, H, self.Hk, self.D, self.bs, self.nb, self.width, self.q.data_ptr(), c[0].data_ptr(),
                                c[1].data_ptr(), s[0].data_ptr(), s[1].data_ptr(), t.data_ptr(), st.data_ptr(), ln.data_ptr(), out.data_ptr(),
                                self.scale_qk, causal, workspace.data_ptr(), workspace.numel(), lse=z.data_ptr() if lse else None, q_stride=self.qs,
                                out_stride=self.os, stream=torch.cuda.current_stream().cuda_stream)
        _sync(backend)
        assert (out[:, H * self.D:] == 7.0).all()                     # between the rows
        return out[:, :H * self.D].double().cpu().numpy().reshape(self.rows, H, self.D), z.double().cpu().numpy()

    def check(self, out, lse, causal=True):
        H, last = self.Hk * self.G, int(self.starts[-1])
        q = self.q[:, :H * self.D].double().cpu().numpy().reshape(self.rows, H, self.D)
        want, wlse, mag = kv_oracle.attend(q, self.codes[0], self.codes[1], self.scale[0], self.scale[1], self.table, self.starts, self.lens,
                                           self.scale_qk, causal, self.G)
        assert (out[last:] == 7.0).all() and (lse[last:] == 7.0).all()               # rows behind the last request
        out, lse, want, wlse, mag = out[:last], lse[:last], want[:last], wlse[:last], mag[:last]
        eps = {BF16: 2.0 ** -8, F16: 2.0 ** -11}[self.dtype]
        largest = np.nanmax(np.abs(kv_oracle.VALUES[:127])) * self.scale[1].max()
        tol = eps * np.abs(want) + (2.0 ** -11 + 2.0 ** -18) * mag + self.lens.max() * 2.0 ** -25 * largest + 1e-30
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(out), nan), "NaN in other places"
        worst = np.where(nan, 0.0, np.abs(out - want) / tol).max() if out.size else 0.0
        assert worst <= 1.0, f"error is {worst:.2f} of the tolerance"
        inf = np.isinf(wlse)
        assert np.array_equal(np.isinf(lse), inf) and np.array_equal(np.isnan(lse), np.isnan(wlse))
        # scores are sums of D products in fp32 (each within 2^-24 of the sum of magnitudes, itself under 2^7): 2^-15 covers them
        assert np.nanmax(np.where(inf, 0.0, np.abs(np.where(inf, 0, lse) - np.where(inf, 0, wlse))), initial=0.0) <= 2.0 ** -15
        return worst


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("context, new, Hk, G, bs", [
    ([0], [1], 1, 1, 16), ([0, 1, 14, 15, 16, 17], [1] * 6, 2, 1, 16), ([500, 3, 129], [1, 1, 1], 2, 4, 16), ([31, 32, 63, 64, 300], [1] * 5, 1, 8, 32),
    ([1000], [1], 1, 3, 64), ([127, 128, 129, 255], [1] * 4, 2, 5, 128), ([700, 90], [1, 1], 1, 16, 16), ([333], [1], 1, 32, 16), ([90], [1], 1, 71, 16)])
def test_attention_of_single_tokens(backend, dtype, D, context, new, Hk, G, bs):
    b = Batch(context, new, Hk, G, D, bs, dtype, seed=D + G)
    b.check(*b.run(backend))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("context, new, Hk, G, bs", [
    ([20, 0, 100], [4, 2, 7], 2, 1, 16), ([64, 5], [8, 8], 1, 4, 32), ([0], [33], 2, 2, 16), ([17, 200, 0], [40, 1, 19], 1, 5, 16), ([0, 30], [130, 70], 2, 4, 64),
    ([250], [129], 1, 8, 128), ([3], [257], 1, 1, 16), ([0], [1], 1, 1, 64), ([600], [64], 1, 3, 32)])
def test_attention_of_several_tokens_and_chunks(backend, dtype, D, causal, context, new, Hk, G, bs):
    b = Batch(context, new, Hk, G, D, bs, dtype, seed=D + G + causal)
    b.check(*b.run(backend, causal), causal)


@pytest.mark.parametrize("G, new", [(1, [1, 1, 1, 1]), (4, [3, 1, 0, 2]), (4, [40, 1, 0, 60])])
def test_attention_of_requests_without_keys_or_queries(backend, G, new):
    b = Batch([0, 50, 40, 0], new, 2, G, 64, 16, BF16, seed=3)
    b.lens[3] = 0                                                     # queries, but not one key
    b.check(*b.run(backend))
    b.check(*b.run(backend, causal=False), causal=False)
    b = Batch([0, 0], [0, 0], 2, G, 64, 16, BF16, seed=3)             # nothing at all
    b.check(*b.run(backend, max_query=5))


@pytest.mark.parametrize("n, length", [(5, 3), (100, 40), (200, 199)])
def test_causal_rows_before_the_first_key_see_nothing(backend, n, length):
    b = Batch([0, 30], [n, 2], 2, 2, 128, 16, BF16, seed=5)
    b.lens[0] = length
    out, lse = b.run(backend)
    b.check(out, lse)
    assert (out[:n - length] == 0).all() and np.isneginf(lse[:n - length]).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [6, 2, 3], [70, 40, 129]])
def test_attention_masks_blocks_outside_the_pool(backend, new):
    b = Batch([100, 64, 10], new, 2, 4, 64, 16, BF16, seed=8)
    b.table[0, 2], b.table[0, 5], b.table[1, 0], b.table[2, :] = -1, b.nb, 2 ** 31 - 1, -2 ** 31
    b.check(*b.run(backend))
    b.check(*b.run(backend, causal=False), causal=False)


@pytest.mark.parametrize("new", [[1, 1], [7, 3], [90, 140]])
def test_attention_reads_strided_queries_and_writes_strided_rows(backend, new):
    b = Batch([75, 200], new, 2, 4, 128, 16, F16, seed=9, q_stride=8 * 128 * 3, out_stride=8 * 128 + 8, width=40)
    b.check(*b.run(backend, lse=True))
    out, lse = b.run(backend, lse=False)
    assert (lse == 7.0).all()


@pytest.mark.parametrize("new", [[3, 4], [50, 90]])
def test_nan_reaches_only_the_rows_that_see_it(backend, new):
    """A NaN value in a token that some rows of the chunk do not see yet, and a NaN key."""
    b = Batch([20, 33], new, 2, 2, 64, 16, BF16, seed=10)
    def put(which, r, pos, d):
        b.codes[which, b.table[r, pos // 16], 1, pos % 16, d] = 0xff
    put(1, 0, 20 + new[0] - 2, 7)
    put(0, 1, 33 + new[1] - 1, 3)
    out, lse = b.run(backend)
    b.check(out, lse)
    assert np.isnan(out).any() and np.isnan(lse).any()


def test_nan_and_infinite_queries_stay_in_their_rows(backend):
    for new in ([1, 3], [60, 80]):
        b = Batch([40, 80], new, 2, 2, 64, 16, BF16, seed=11)
        b.q[1, 70] = float("nan")
        b.q[2, 5] = float("inf")
        out, lse = b.run(backend)
        H = 4
        for row, h in ((1, 70 // 64), (2, 0)):
            assert np.isnan(out[row, h]).all() and np.isnan(lse[row, h])
            out[row, h], lse[row, h] = 7.0, 7.0
        b.q[1:3] = 0
        keep = np.ones((b.rows, H), bool)
        keep[1, 1] = keep[2, 0] = False
        q = b.q.double().cpu().numpy().reshape(b.rows, H, 64)
        assert np.isfinite(out[keep]).all()


@pytest.mark.parametrize("new", [[1], [5], [130]])
def test_scales_that_differ_widely_between_blocks(backend, new):
    """A block of tiny values that gets nearly all the weight beside blocks of large ones (and the other way round)."""
    b = Batch([200], new, 1, 2, 64, 16, BF16, seed=12, sharp=3.0)
    b.scale[1, b.table[0, :5]] = 2.0 ** -30
    b.scale[1, b.table[0, 5]] = 2.0 ** 20
    b.scale[0, b.table[0, 3]] = 2.0 ** -3                             # large keys: sharp softmax
    out, lse = b.run(backend)
    b.check(out, lse)


@pytest.mark.parametrize("G", [1, 4])
def test_small_values_keep_their_digits_beside_an_all_but_masked_block(backend, G):
    """All the weight on a block whose values are 2^-24 of another's: the result is as exact as if the other were not there."""
    b = Batch([31], [1], 1, G, 64, 16, F16, seed=13)
    keys = np.zeros((16, 64))
    keys[:, 0] = 448.0
    b.codes[0, b.table[0, 0], 0], b.codes[0, b.table[0, 1], 0] = kv_oracle.encode(keys), kv_oracle.encode(-keys)
    b.scale[0, b.table[0]] = 2.0 ** -5
    b.q[:, ::64] = 16.0
    b.scale[1, b.table[0, 0]], b.scale[1, b.table[0, 1]] = 2.0 ** -8, 2.0 ** 16
    out, lse = b.run(backend)
    q = b.q.double().cpu().numpy().reshape(b.rows, G, 64)
    want, _, mag = kv_oracle.attend(q, b.codes[0], b.codes[1], b.scale[0], b.scale[1], b.table, b.starts, b.lens, b.scale_qk, True, G)
    assert (np.abs(out[:1] - want[:1]) <= 2.0 ** -11 * np.abs(want[:1]) + (2.0 ** -11 + 2.0 ** -14) * mag[:1]).all()


@pytest.mark.parametrize("context, new, G", [([40000], [1], 4), ([30000, 5, 9000], [1, 1, 1], 1), ([9000], [6], 4), ([12000, 100], [70, 1], 2)])
def test_long_sequences_are_split_and_joined(backend, context, new, G):
    b = Batch(context, new, 2, G, 64, 64, BF16, seed=14)
    first = b.run(backend)
    b.check(*first)
    again = b.run(backend)
    assert all(np.array_equal(x, y) for x, y in zip(first, again))    # the same bits each time


def test_many_short_requests(backend):
    rng = np.random.default_rng(15)
    b = Batch(rng.integers(0, 90, 700).tolist(), rng.integers(0, 4, 700).tolist(), 1, 2, 64, 16, BF16, seed=15)
    b.check(*b.run(backend))


@pytest.mark.parametrize("dtype, D, G, bs", [(BF16, 64, 8, 16), (F16, 128, 8, 32), (BF16, 128, 16, 128)])
def test_many_chunks_of_one_and_two_tiles(backend, dtype, D, G, bs):
    """More items than CTAs: each walks several, of 33 to 320 rows in any order, with requests of few rows and of none between."""
    rng = np.random.default_rng(D + G)
    new = [int(x) for x in rng.choice([0, 1, 2, 5, 9, 16, 17, 20], 260)]
    context = [int(x) for x in rng.choice([0, 1, 30, 70, 200], 260)]
    b = Batch(context, new, 2, G, D, bs, dtype, seed=G)
    b.check(*b.run(backend))


def test_a_request_longer_than_its_table_row_counts_as_that_long(backend):
    b = Batch([60], [4], 2, 2, 64, 16, BF16, seed=16)
    b.lens[0] = 1 << 30
    out, lse = b.run(backend, causal=False)
    b.check(out, lse, causal=False)


@pytest.mark.parametrize("new", [[1, 1], [4, 9], [100, 30]])
def test_workspace_is_left_ready_for_the_next_call(backend, new):
    """Calls of different shapes, one after the other with one workspace, and graphs that share it."""
    torch = _torch()
    big, small = Batch([5000, 900], new, 2, 4, 128, 16, BF16, seed=17), Batch([70, 3000], new, 1, 2, 64, 32, F16, seed=18)
    ws = torch.zeros(max(backend.paged_attention_workspace_bytes(2, max(new), 8, 2, 128), backend.paged_attention_workspace_bytes(2, max(new), 2, 1, 64)),
                     dtype=torch.uint8, device="cuda")
    for _ in range(3):
        big.check(*big.run(backend, workspace=ws))
        small.check(*small.run(backend, workspace=ws))


def test_offsets_beyond_four_gigabytes(backend):
    torch = _torch()
    nb, Hk, bs, D = 17000, 8, 128, 128                                # 2.2 GB of keys and as much of values; a token's row lies past 2^31
    k, v = (torch.zeros((2 * nb, Hk, bs, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones((2 * nb, Hk), device="cuda") for _ in range(2))
    b = Batch([250, 100], [1, 40], Hk, 2, D, bs, BF16, seed=19)
    ids = np.array([2 * nb - 1, 2 * nb - 3, nb - 1, 2 * nb - 2, 5, nb + 1, nb + 5, 77])[:b.nb]
    assert b.nb <= len(ids)
    at = _dev(ids)
    for dst, src in ((k, b.codes[0]), (v, b.codes[1])):
        dst[at] = _dev(src)
    ks[at], vs[at] = _dev(b.scale[0]), _dev(b.scale[1])
    table = np.where(b.table >= 0, ids[np.maximum(b.table, 0)], -1).astype(np.int32)
    ws = torch.zeros(backend.paged_attention_workspace_bytes(2, 40, 16, 8, D), dtype=torch.uint8, device="cuda")
    out = torch.full((b.rows, b.os), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((b.rows, 16), 7.0, device="cuda")
    t, st, ln = _dev(table), _dev(b.starts), _dev(b.lens)
    stream = torch.cuda.current_stream().cuda_stream
    backend.paged_attention(BF16, 2, 40, 16, Hk, D, bs, 2 * nb, table.shape[1], b.q.data_ptr(), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(),
                            t.data_ptr(), st.data_ptr(), ln.data_ptr(), out.data_ptr(), b.scale_qk, True, ws.data_ptr(), ws.numel(), lse=lse.data_ptr(), stream=stream)
    _sync(backend)
    b.check(out.double().cpu().numpy().reshape(b.rows, 16, D), lse.double().cpu().numpy())
    # and the write: the last block of the pool
    x = torch.randn((3, Hk * D), device="cuda").to(torch.bfloat16)
    slots = _dev(np.array([(2 * nb - 1) * bs + i for i in range(3)], np.int64))
    backend.kv_write(BF16, 3, Hk, D, bs, 2 * nb, x.data_ptr(), x.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), stream=stream)
    _sync(backend)
    codes, scale = np.zeros((1, Hk, bs, D), np.uint8), np.ones((1, Hk))
    kv_oracle.write(x.double().cpu().numpy().reshape(3, Hk, D), [0, 1, 2], codes, scale)
    assert np.array_equal(k[-1, :, :3].cpu().numpy(), codes[0, :, :3]) and np.array_equal(ks[-1].cpu().numpy(), scale[0])
