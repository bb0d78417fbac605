"""The decode step over the 8-bit paged cache against a CPU restatement: decode_ref's step with the cache of kv8_ref."""
import ctypes

import numpy as np
import pytest

import oracle
from demonic_b200 import _lib, decoder
from tests import kv8_ref
from tests.parity import TOL_BF16, scaled_err

pytestmark = pytest.mark.gpu
F = np.float32
CFG = decoder.Config(layers=2, d_model=256, heads=2, head_dim=128, ffn=520, vocab=1003, max_len=70)


@pytest.fixture(autouse=True)
def clean():
    _lib.load().dmc_cuda_clear_error()
    yield
    _lib.load().dmc_cuda_clear_error()


def ref_step(cfg, model, books: kv8_ref.Model, seq: int, token: int):
    """One step of sequence `seq` (tests/decode_ref.py, with the cache quantised); the logits."""
    d, h, hd, f = cfg.d_model, cfg.heads, cfg.head_dim, cfg.ffn
    assert books.reserve([seq], [1])
    pos = int(books.lens[seq]) - 1
    x = oracle.embed_bf16(model["embed"], token)
    cs, sn = model["rope_cos"][pos], model["rope_sin"][pos]
    for i, L in enumerate(model["layers"]):
        xn = oracle.rms_norm_f32(x, L["gain1"], cfg.eps)
        qkv = oracle.gemm_bf16_nt(xn.reshape(1, d), L["wqkv"])[0]
        q, k, v = (qkv[j * d:(j + 1) * d].reshape(h, hd).copy() for j in range(3))
        for j in range(h):
            q[j], k[j] = oracle.rope_row(q[j], cs, sn), oracle.rope_row(k[j], cs, sn)
        books.append(i, k.reshape(1, 1, h, hd), v.reshape(1, 1, h, hd), [seq], 1)
        ao, _, _ = books.attention(i, q.reshape(1, 1, h, hd).astype(np.float64), [seq], hd ** -0.5)
        x = x + oracle.gemm_bf16_nt(ao.reshape(1, d).astype(F), L["wo"])[0]
        xn = oracle.rms_norm_f32(x, L["gain2"], cfg.eps)
        gu = oracle.gemm_bf16_nt(xn.reshape(1, d), L["wgu"])[0]
        act = (oracle.silu(gu[:f]) * gu[f:]).astype(F)
        x = x + oracle.gemm_bf16_nt(act.reshape(1, f), L["wd"])[0]
    xn = oracle.rms_norm_f32(x, model["gain_final"], cfg.eps)
    return oracle.gemm_bf16_nt(xn.reshape(1, d), model["lm_head"])[0]


def test_sequences_that_are_stepped_forked_released_and_compacted():
    cfg = CFG
    model = decoder.random_model(cfg, seed=3, cache_len=0)
    dec = decoder.Kv8Decoder(cfg, model, sequences=3, pages=11, page_tokens=16)
    books = kv8_ref.Model(cfg.layers, 11, cfg.heads, 16, cfg.head_dim, 3, -(-cfg.max_len // 16))
    rng = np.random.default_rng(8)

    def both(seq, token, **how):
        u = float(F(rng.random()))
        nxt, prob, logits = dec.step(seq, token, u=u, want_logits=True, **how)
        want = ref_step(cfg, model, books, seq, token)
        # a K or V next to a rounding border may fall to the other side of it: the bar of bf16 weights, not elementwise
        assert scaled_err(logits, want) <= TOL_BF16
        t, p = kv8_ref.sample_row(logits, how.get("temperature", 0.0), how.get("top_k", 0), how.get("top_p", 1.0),
                                  how.get("min_p", 0.0), u)
        assert nxt == t and abs(prob - p) <= p * 1e-6
        assert dec.length(seq) == books.lens[seq] and dec.free_pages == books.count
        return nxt

    token = 5
    for i in range(21):                                   # over a page border
        token = both(0, token, temperature=0.9, top_k=50, top_p=0.9) if i % 3 else both(0, token)
    dec.fork(0, 1)
    books.fork([0], [1])
    a, b = token, (token + 1) % cfg.vocab
    for _ in range(14):                                   # each writes into its own copy, and on to a new page
        a, b = both(0, a, temperature=0.7, min_p=0.05), both(1, b, temperature=1.3)
    both(2, 7)
    dec.release(0)
    books.release([0])
    dec.compact()
    books.compact()
    assert dec.length(0) == 0 and dec.free_pages == books.count
    for _ in range(3):
        b = both(1, b)
    both(0, 1002)
    dec.close()
    assert _lib.load().dmc_cuda_status() == 0


def test_a_fork_continues_with_the_same_bits():
    model = decoder.random_model(CFG, seed=4, cache_len=0)
    dec = decoder.Kv8Decoder(CFG, model, sequences=2)
    for t in (3, 9, 27, 81):
        dec.step(0, t)
    dec.fork(0, 1)
    a = dec.step(0, 100, want_logits=True)[2]
    b = dec.step(1, 100, want_logits=True)[2]
    assert np.array_equal(a, b)
    dec.close()


def test_without_a_page_left_the_sequence_stays_as_it_was():
    model = decoder.random_model(CFG, seed=5, cache_len=0)
    dec = decoder.Kv8Decoder(CFG, model, sequences=2, pages=2, page_tokens=16)
    for t in range(16):
        dec.step(0, t)
    dec.step(1, 1)
    with pytest.raises(_lib.DmcCudaError) as e:
        dec.step(0, 77)
    assert e.value.code == 4 and "no page is left" in str(e.value)
    _lib.load().dmc_cuda_clear_error()
    assert dec.length(0) == 16 and dec.free_pages == 0
    dec.release(1)
    got = dec.step(0, 77, want_logits=True)[2]
    other = decoder.Kv8Decoder(CFG, model, sequences=1)
    for t in range(16):
        other.step(0, t)
    assert np.array_equal(got, other.step(0, 77, want_logits=True)[2])
    other.close()
    dec.close()


def test_refusals():
    lib = _lib.load()
    model = decoder.random_model(CFG, seed=6, cache_len=0)
    dec = decoder.Kv8Decoder(CFG, model, sequences=2)
    plain = decoder.Decoder(CFG, decoder.random_model(CFG, seed=6, cache_len=0))

    def refused(call, code, text):
        call()
        assert lib.dmc_cuda_status() == code and text in lib.dmc_cuda_last_error().decode()
        lib.dmc_cuda_clear_error()
    h, p = dec.handle, plain.handle
    refused(lambda: lib.dmc_decoder_step_kv8(h, 2, 0, None, None, None, None), 2, "sequence 2 of 2")
    refused(lambda: lib.dmc_decoder_step_kv8(p, 0, 0, None, None, None, None), 2, "not a decoder with an 8-bit cache")
    refused(lambda: lib.dmc_decoder_step(h, 0, 0, None, None), 2, "dmc_decoder_step_kv8")
    refused(lambda: lib.dmc_decoder_fork(h, 0, 0), 2, "decoder_fork")
    dec.step(1, 1)
    refused(lambda: lib.dmc_decoder_fork(h, 0, 1), 2, "has to be empty")
    refused(lambda: lib.dmc_decoder_release(h, -1), 2, "decoder_release")
    assert lib.dmc_decoder_bench(h, 0, 5, 1, 0) == -1.0
    lib.dmc_cuda_clear_error()
    dec.step(0, 1)
    assert dec.bench(1, 0, 3) > 0
    with pytest.raises(_lib.DmcCudaError):
        decoder.Kv8Decoder(CFG, model, page_tokens=8)
    lib.dmc_cuda_clear_error()
    for _ in range(CFG.max_len - 1):
        dec.step(1, 1)
    refused(lambda: lib.dmc_decoder_step_kv8(h, 1, 0, None, None, None, None), 2, "is full")
    dec.close()
    plain.close()


def test_the_benchmark_writes_to_no_page_that_another_sequence_holds():
    model = decoder.random_model(CFG, seed=7, cache_len=0)
    dec = decoder.Kv8Decoder(CFG, model, sequences=2)
    for t in (3, 4, 5):
        dec.step(0, t)
    dec.fork(0, 1)
    with pytest.raises(_lib.DmcCudaError) as e:
        dec.bench(6, 2, 1)
    assert e.value.code == 2 and "another sequence" in str(e.value)
    _lib.load().dmc_cuda_clear_error()
    dec.step(0, 6)                              # (its last page is its own now)
    assert dec.bench(7, 3, 1) > 0
    got = dec.step(1, 6, want_logits=True)[2]
    other = decoder.Kv8Decoder(CFG, model)
    for t in (3, 4, 5):
        other.step(0, t)
    assert np.array_equal(got, other.step(0, 6, want_logits=True)[2])
    other.close()
    dec.close()


@pytest.mark.parametrize("held", [16, 32])
@pytest.mark.parametrize("way", [(0, 1), (1, 0)], ids=["from", "to"])
def test_the_benchmark_is_refused_where_a_full_last_page_is_shared(held, way):
    model = decoder.random_model(CFG, seed=8, cache_len=0)
    dec = decoder.Kv8Decoder(CFG, model, sequences=2, page_tokens=16)
    for t in range(held):
        dec.step(way[0], t)
    dec.fork(*way)
    with pytest.raises(_lib.DmcCudaError) as e:
        dec.bench(999, held - 1, 1)             # would replace the last token of the page that both hold
    assert e.value.code == 2 and "another sequence" in str(e.value)
    _lib.load().dmc_cuda_clear_error()
    dec.step(0, 6)                              # a page of its own
    assert dec.bench(7, held, 1) > 0
    got = dec.step(1, 6, want_logits=True)[2]
    other = decoder.Kv8Decoder(CFG, model)
    for t in range(held):
        other.step(0, t)
    assert np.array_equal(got, other.step(0, 6, want_logits=True)[2])
    other.close()
    dec.close()


@pytest.mark.parametrize("kv8", [True, False], ids=["kv8", "f32"])
def test_a_decoder_that_does_not_fit_leaves_no_memory_behind(kv8):
    lib, rt = _lib.load(), ctypes.CDLL("libcudart.so.12")
    rt.cudaMemGetInfo.argtypes = [ctypes.POINTER(ctypes.c_size_t)] * 2
    # embeddings of 128 MiB and activations of 3 GiB fit; the first layer's gate and up matrices, 256 GiB, do not
    desc = _lib.DecoderConfig(2, 256, 2, 128, 1 << 28, 262144, 64, 1e-5)

    def create():
        out = ctypes.c_void_p()
        rc = (lib.dmc_decoder_create_kv8(ctypes.byref(desc), 2, 64, 16, ctypes.byref(out)) if kv8
              else lib.dmc_decoder_create(ctypes.byref(desc), ctypes.byref(out)))
        assert rc == 4 and not out.value
        lib.dmc_cuda_clear_error()
        free, total = ctypes.c_size_t(), ctypes.c_size_t()
        assert rt.cudaMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
        return free.value
    first = create()                              # (the context and its first buffers are made on the way)
    assert [create() for _ in range(3)] == [first] * 3
    small = decoder.Kv8Decoder(CFG, decoder.random_model(CFG, seed=9, cache_len=0))
    assert small.step(0, 3)[1] == 1.0
    small.close()


def test_a_large_pool_starts_with_every_page_free():
    """Zeroing 30 GiB takes milliseconds, in which the free stack is written already."""
    pages = 1_900_000
    dec = decoder.Kv8Decoder(CFG, decoder.random_model(CFG, seed=10, cache_len=0), sequences=2, pages=pages)
    assert dec.free_pages == pages
    for t in range(17):
        dec.step(0, t)
    assert dec.free_pages == pages - 2
    dec.release(0)
    assert dec.free_pages == pages
    dec.close()
