"""Sampling on the device against its definition in 64 bits (tests/kv8_ref.py)."""
import numpy as np
import pytest

from demonic_b200 import _lib, backend, sampling
from demonic_b200.backend import DeviceBuffer
from demonic_b200.synth import bf16_to_f32, f32_to_bf16_rne
from tests import kv8_ref

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.fixture(autouse=True)
def clean():
    _lib.load().dmc_cuda_clear_error()
    yield
    assert _lib.load().dmc_cuda_status() == 0


def check(x, t, k, p, mp, u, bits=None, stride=None):
    """x: [batch, vocab] f32; every filter an array or None."""
    batch, vocab = x.shape
    stride = stride or vocab
    src = bits if bits is not None else x
    rows = np.zeros((batch, stride), src.dtype)
    rows[:, :vocab] = src
    rows[:, vocab:] = 0x7F00 if bits is not None else 1e30        # behind a row: would win everything
    dev = {n: None if a is None else DeviceBuffer.from_host(np.asarray(a, np.int32 if n == "top_k" else F))
           for n, a in (("temperature", t), ("top_k", k), ("top_p", p), ("min_p", mp))}
    tokens, prob = DeviceBuffer.from_host(np.full(batch + 1, 77, np.int32)), DeviceBuffer(batch * 4)
    sampling.sample(DeviceBuffer.from_host(rows), batch, vocab, tokens, DeviceBuffer.from_host(np.asarray(u, F)), prob=prob,
                    row_stride=stride, xdtype="bf16" if bits is not None else "f32", **dev)
    backend.sync()
    got, pr = tokens.download(np.int32, batch + 1), prob.download(F, batch)
    assert got[batch] == 77
    for r in range(batch):
        at = lambda a, none: none if a is None else (np.asarray(a, F)[r].item() if a is not k else int(a[r]))  # noqa: E731
        want, wp = kv8_ref.sample_row(x[r], at(t, 1.0), at(k, 0), at(p, 1.0), at(mp, 0.0), float(F(u[r])))
        assert got[r] == want, f"row {r}: token {got[r]}, {want} expected"
        # prob: one rounding to f32, and masses off by half a unit of 2^-44 per member of a whole of at least 1
        assert abs(pr[r] - wp) <= wp * (2.0 ** -24 + vocab * 2.0 ** -44) + 1e-30
    return got[:batch]


@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1000, 4097, 32000, 50257, 128000, 262144])
@pytest.mark.parametrize("kind", ["none", "k", "p", "kp", "mp", "all"])
def test_filters_and_vocabularies(vocab, kind):
    rng = np.random.default_rng(vocab)
    batch = 9 if vocab < 40000 else 3
    x = (rng.standard_normal((batch, vocab)) * 2.5).astype(F)
    x[:, rng.integers(0, vocab, 5)] += 6
    t = rng.uniform(0.4, 1.5, batch)
    k = rng.integers(1, 80, batch) if kind in ("k", "kp", "all") else None
    p = rng.uniform(0.3, 0.999, batch) if kind in ("p", "kp", "all") else None
    mp = rng.uniform(0.001, 0.3, batch) if kind in ("mp", "all") else None
    u = rng.random(batch)
    u[0] = 0.0
    u[-1] = np.float32(1) - np.float32(2.0 ** -24)
    check(x, t, k, p, mp, u)


@pytest.mark.parametrize("vocab,stride", [(50257, 50257), (513, 520), (1000, 1003), (31, 33)])
def test_bf16_rows_that_start_anywhere(vocab, stride):
    rng = np.random.default_rng(vocab)
    bits = f32_to_bf16_rne(rng.standard_normal((6, vocab)) * 3)
    x = bf16_to_f32(bits).reshape(6, vocab)      # (bf16: many equal logits)
    check(x, rng.uniform(0.5, 1.2, 6), [0, 5, 50, 0, 17, 3], [1, .9, .5, .95, 1, .2], [0, 0, .1, 0, .02, 0], rng.random(6),
          bits=bits, stride=stride)
    check(x, None, None, None, None, rng.random(6), bits=bits, stride=stride)
    check(x, None, None, [.999] * 6, None, rng.random(6), bits=bits, stride=stride)


def test_greedy_ties_and_empty_rows():
    x = np.zeros((8, 300), F)
    x[0, 40] = x[0, 250] = 3.0
    x[1] = -np.inf
    x[2] = np.nan
    x[3] = np.nan
    x[3, 123] = -5.0
    x[4] = -np.inf
    x[4, 17] = -np.inf
    x[4, 200] = np.finfo(F).min
    x[5, [3, 250]] = np.inf
    x[6] = np.finfo(F).min
    x[7, 5] = -0.0
    zero = np.zeros(8)
    got = check(x, zero, None, None, None, zero)
    assert got.tolist() == [40, -1, -1, 123, 200, 3, 0, 0]
    check(x, np.full(8, -1.0), None, None, None, zero)
    check(x, np.full(8, np.nan), None, None, None, zero)
    for u in (0.0, 0.3, 0.7, 0.99):
        for k, p in ((None, None), ([2] * 8, None), (None, [0.5] * 8), ([100] * 8, [0.25] * 8)):
            check(x, np.full(8, 0.8), k, p, None, np.full(8, u))


def test_rows_of_equal_values_and_masked_rows():
    rng = np.random.default_rng(1)
    vocab = 20000
    x = np.zeros((6, vocab), F)
    x[1] = np.finfo(F).min                        # a mask of the type's lowest value
    x[1, 500:700] = rng.standard_normal(200)
    x[2] = -np.inf
    x[2, ::7] = 1.0
    x[3, 9000:] = 1e-6                            # two values next to one another
    x[4] = rng.integers(0, 3, vocab)
    x[5, 77] = 40.0                               # one far above the rest, which have no mass left
    u = rng.random(6)
    check(x, None, None, None, None, u)
    check(x, None, [1500, 30, 2000, 15000, 9000, 5], None, None, u)
    check(x, None, None, [.3, .9, .7, .8, .55, .999999], None, u)
    check(x, None, [15000] * 6, [.5] * 6, [0.5] * 6, u)
    check(x, np.full(6, 1e-20), [5] * 6, [.5] * 6, None, u)
    check(x, np.full(6, 1e20), [50] * 6, [.5] * 6, None, u)
    check(x, np.full(6, np.inf), None, [.5] * 6, None, u)


def test_parameters_out_of_range_are_no_filter():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 777)).astype(F)
    u = rng.random(5)
    a = check(x, None, [0, -3, 777, 778, 2 ** 31 - 1], [1, 1.5, np.nan, np.inf, 2], [0, -1, np.nan, -np.inf, 0], u)
    assert np.array_equal(a, check(x, None, None, None, None, u))
    check(x, None, None, [0, -1, 1e-9, 0, 0], None, u)                 # at least one is kept
    check(x, None, None, None, [2, 1, 5, np.inf, 1], u)
    check(x, None, None, None, None, [1.0, 2.0, 7.0, 1.0, 3.0])        # the last


def test_u_walks_through_the_distribution():
    """The tokens of evenly spread u come in the order of the indices, as often as their probability says."""
    x = np.log(np.array([[0.1, 0.2, 0.3, 0.15, 0.25]])).astype(F)
    n = 400
    u = (np.arange(n) + 0.5) / n
    got = check(np.repeat(x, n, 0), None, None, None, None, u)
    assert np.all(np.diff(got) >= 0)
    assert np.array_equal(np.bincount(got), (np.array([0.1, 0.2, 0.3, 0.15, 0.25]) * n).round())


@pytest.mark.parametrize("batch,vocab", [(593, 40), (1024, 61), (1025, 33), (90, 20001)])
@pytest.mark.parametrize("kind", ["mixed", "all_slow", "k_alone"])
def test_batches_that_do_not_fit_at_once(batch, vocab, kind):
    """Slow rows are taken first: every row still gets its own answer, whichever cluster takes it."""
    rng = np.random.default_rng(batch)
    x = (rng.standard_normal((batch, vocab)) * 2).astype(F)
    k = np.where(rng.random(batch) < 0.5, rng.integers(1, vocab, batch), 0) if kind != "all_slow" else None
    p = {"mixed": np.where(rng.random(batch) < 0.5, rng.uniform(0.2, 0.95, batch), 1.0), "all_slow": np.full(batch, 0.8),
         "k_alone": None}[kind]
    t = np.where(rng.random(batch) < 0.1, 0.0, rng.uniform(0.5, 1.5, batch))
    check(x, t, k, p, None, rng.random(batch))


def close_beside_a_large_one(kind, vocab, rng):
    """One logit far above the rest, whose differences are lost in their distance from it (an f32)."""
    if kind == "normal":
        x = rng.standard_normal(vocab) * 1e-7
    elif kind == "every size":                    # from 1e-8 down to below the smallest normal number, both signs, zeros
        x = rng.choice([-1.0, 1.0], vocab) * 10.0 ** rng.uniform(-44, -8, vocab)
        x[::50] = 0.0
        x[1::50] = -0.0
    else:                                         # neighbouring floats, each of them many times
        x = np.float32(1e-6).view(np.int32) + rng.integers(0, 40, vocab).astype(np.int32)
        x = x.view(F).astype(np.float64)
    x[vocab // 3] = 20.0
    return x.astype(F)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["normal", "every size", "neighbours"])
@pytest.mark.parametrize("t", [1.0, 10.0])
@pytest.mark.parametrize("k,p", [(50, None), (600, None), (1000, None), (20000, None), (None, 0.3), (None, 0.9), (900, 0.6), (20000, 0.8)])
def test_logits_closer_together_than_their_distance_from_the_largest(bf16, kind, t, k, p):
    rng = np.random.default_rng(31)
    x = close_beside_a_large_one(kind, 32000, rng)
    bits = None
    if bf16:
        bits = f32_to_bf16_rne(x)
        x = bf16_to_f32(bits).reshape(x.shape)
    n = 12
    rows = np.repeat(x[None], n, 0)
    check(rows, np.full(n, t), None if k is None else [k] * n, None if p is None else [p] * n, None, (np.arange(n) + 0.5) / n,
          bits=None if bits is None else np.repeat(bits.reshape(1, -1), n, 0))


def test_largest_rows_that_do_not_fit_at_once():
    """An f32 slice of 128 KiB fills an SM, so that 19 rows and more are taken in the order of their cost."""
    rng = np.random.default_rng(77)
    batch, vocab = 21, 262144
    x = (rng.standard_normal((batch, vocab)) * 2).astype(F)
    i = np.arange(batch)
    check(x, np.full(batch, 0.8), np.where(i % 3 == 1, 50, 0), np.where(i % 3 == 2, 0.9, 1.0), None, rng.random(batch))


def test_a_logit_beyond_the_range_of_f32_below_the_largest_is_never_drawn():
    x = np.full((4, 100), -3e38, F)
    x[:, 7] = 3e38
    for k, p in ((None, None), ([5] * 4, None), (None, [0.9] * 4)):
        u, tokens, prob = DeviceBuffer.from_host(np.array([0, .4, .9, .999], F)), DeviceBuffer(16), DeviceBuffer(16)
        dev = {n: None if a is None else DeviceBuffer.from_host(np.asarray(a, np.int32 if n == "top_k" else F))
               for n, a in (("top_k", k), ("top_p", p))}
        sampling.sample(DeviceBuffer.from_host(x), 4, 100, tokens, u, temperature=DeviceBuffer.from_host(np.full(4, np.inf, F)),
                        prob=prob, **dev)
        backend.sync()
        assert tokens.download(np.int32, 4).tolist() == [7] * 4 and prob.download(F, 4).tolist() == [1.0] * 4
