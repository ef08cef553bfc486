"""Batched decode with the cross-attention K/V in 4-bit pages (ms_options.cross_kv_bits = 4)
against the CPU oracle whose stored cross K/V are quantized by the definition."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
from moonshine_b200 import synth  # noqa: E402
from test_batch_gpu import _check_batch  # noqa: E402
from util import BF16_LOGIT_TOL, FP32_LOGIT_TOL, model_dir, oracle_for  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture
def oracle4(monkeypatch):
    """The oracle's decoder caches hold the cross K/V that the 4-bit codes stand for."""
    from oracle.moonshine_oracle import DecoderCache, Oracle

    def new_cache(self, memory, kv_fp16):
        cache = DecoderCache(self, memory, kv_fp16)
        four = lambda x: ref.quantize(torch.from_numpy(np.ascontiguousarray(x)))[3].numpy().astype(x.dtype)  # noqa: E731
        cache.cross_k = [four(x) for x in cache.cross_k32]
        cache.cross_v = [four(x) for x in cache.cross_v32]
        return cache
    monkeypatch.setattr(Oracle, "new_cache", new_cache)


# The engine's K/V differ from the oracle's by its products' rounding, r of a head's range (fp32
# checkpoints: 1e-5 at most, bf16: 2^-8 of each term, 1e-2 at most).  That moves a share of at
# most 2 * 15 r of the codes by one step, 1 / 15 of the range: 2 r of the range on average over
# a query's frames, below the tolerances that the same products have with 16-bit K/V.
def test_fp32_checkpoint(model_root, oracle4):
    import moonshine_b200 as mb
    d = model_dir(model_root, "tiny")
    m = mb.MoonshineModel.load(d, cross_kv_bits=4)
    audios = [synth.synth_audio(n, 900 + i) for i, n in enumerate([16000, 48000, 30000, 1300, 80000])]
    _check_batch(d, audios, 24, model=m, tol=FP32_LOGIT_TOL)
    _check_batch(d, audios[:2], None, model=m, tol=FP32_LOGIT_TOL)  # a smaller call, own limits


def test_bf16_checkpoint(model_root, oracle4):
    import moonshine_b200 as mb
    d = model_dir(model_root, "small", dtype="bfloat16", vocab_size=2048, max_position_embeddings=512)
    m = mb.MoonshineModel.load(d, cross_kv_bits=4)
    audios = [synth.synth_audio(n, 920 + i) for i, n in enumerate([24000, 17777, 32000])]
    _check_batch(d, audios, 8, model=m, tol=BF16_LOGIT_TOL)


def test_stored_rows_are_read_from_the_second_call_on(model_root):
    """The first decoder call reads the fp32 rows; later ones differ from 16-bit storage by the
    quantization, and two runs of one batch give the same bits."""
    import moonshine_b200 as mb
    d = model_dir(model_root, "tiny")
    audios = [synth.synth_audio(n, 940 + i) for i, n in enumerate([32000, 20000])]
    four, sixteen = mb.MoonshineModel.load(d, cross_kv_bits=4), mb.MoonshineModel.load(d)
    _, _, a = four.generate_batch(audios, forced_len=6, return_logits=True)
    _, _, b = sixteen.generate_batch(audios, forced_len=6, return_logits=True)
    assert np.array_equal(a[:, 0], b[:, 0])
    assert not np.array_equal(a[:, 1], b[:, 1])
    ids, _, again = four.generate_batch(audios, forced_len=6, return_logits=True)
    assert np.array_equal(a, again)
    assert ids == four.generate_batch(audios, forced_len=6)[0]  # captured steps and eager ones


def test_other_calls_keep_their_cache(model_root):
    """generate and lockstep streams of a model loaded with 4-bit cross K/V, before and after a
    batch: as those of a model without."""
    import moonshine_b200 as mb
    d = model_dir(model_root, "tiny")
    four, sixteen = mb.MoonshineModel.load(d, cross_kv_bits=4), mb.MoonshineModel.load(d)
    a = synth.synth_audio(48000, 960)

    def streamed(m):
        st = [m.create_stream() for _ in range(2)]
        got = []
        for k in range(3):
            for i, s in enumerate(st):
                if k == 0:
                    m.start_stream(s)
                m.add_audio(s, synth.synth_audio(6400, 970 + 10 * k + i))
            got.append(m.transcribe_batch(st, streaming_config=mb.StreamingConfig(batch_decode=1), max_tokens=8))
        for s in st:
            s.close()
        return got
    want, want_streams = sixteen.generate(a, forced_len=20).tokens, streamed(sixteen)
    for _ in range(2):
        assert four.generate(a, forced_len=20).tokens == want
        assert streamed(four) == want_streams
        four.generate_batch([a, a[:16000]], forced_len=8)


def test_refused_bits(model_root):
    import moonshine_b200 as mb
    with pytest.raises(ValueError, match="cross_kv_bits"):
        mb.MoonshineModel.load(model_dir(model_root, "tiny"), cross_kv_bits=8)
