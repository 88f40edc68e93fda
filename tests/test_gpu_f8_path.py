"""The acoustic model with its dense layers in 8-bit floating point (tunable am_f8 = 1, STTX_GetAcousticMode 2), through the model's own entry points."""
import os

import numpy as np
import pytest
import torch

from conftest import FIX
from stt_amd import blocks, native, synth

pytestmark = pytest.mark.gpu


def _model(tmp_path, w, name, f8=True, beam_width=100):
    from stt_amd import Model, modelfile
    p = str(tmp_path / (name + ".sttw"))
    modelfile.write_model(p, w, synth.ENGLISH_LABELS, beam_width=beam_width)
    native.set_tuning("am_f8", int(f8))
    try:
        m = Model(p)
    finally:
        native.set_tuning("am_f8", 0)
    assert m.acousticMode() == (2 if f8 else 0)
    return m


@pytest.fixture(scope="module")
def small(tmp_path_factory):
    w = synth.synth_weights(31, n_hidden=256)
    w["layer_6/weights"] = (w["layer_6/weights"] * 6.0).astype(np.float32)
    m = _model(tmp_path_factory.mktemp("f8"), w, "small")
    m.enableExternalScorer(os.path.join(FIX, "pruned_lm.scorer"))
    return m, w


def test_probabilities_are_the_operators_own(small):
    """The engine's probabilities are those of stt_amd.blocks' layers around the engine's recurrent step, on the same windows: everything up to layer 5
    the same bits; then 256 products a class summed in 32 bits on either side, a few units of 2^-24 of sums below 16: 1e-4 of a probability's
    logarithm has room for all of it."""
    m, w = small
    B, T, H = 64, 43, 256
    audio = [synth.synth_audio(512 + 320 * (T - 2) + 17 * (i % 5), seed=300 + i) for i in range(B)]
    mfcc = [m.computeMfcc(a) for a in audio]
    assert all(f.shape == (T, 26) for f in mfcc)
    win = np.zeros((T, B, 19, 26), np.float16)                # row t * B + b: the 19 frames around t, zeros outside the utterance
    for b in range(B):
        padded = np.zeros((T + 18, 26), np.float32)
        padded[9:9 + T] = mfcc[b]
        for t in range(T):
            win[t, b] = padded[t:t + 19]
    x = torch.from_numpy(win.reshape(T * B, 494)).cuda()      # 2752 rows: enough for the tiled form, whose sums the engine takes at every size
    W = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in w.items()}
    mat = lambda v: blocks.quantize_blocks(v.t().contiguous(), 128)
    for k in ("1", "2", "3"):
        x = blocks.dense_blocks(x, mat(W["layer_%s/weights" % k]), W["layer_%s/bias" % k], relu_clip=20.0, dtype=torch.float8_e4m3fn)
    kernel, bias = w["lstm/kernel"], W["lstm/bias"]
    xproj = blocks.dense_blocks(x, mat(torch.from_numpy(np.ascontiguousarray(kernel[:H])).cuda()), bias, dtype=torch.float32)
    _, _, h_all = m.lstmSteps(xproj.cpu().numpy(), B, T)
    h = torch.from_numpy(h_all.view(np.float16)).cuda()
    y5 = blocks.dense_blocks(h, mat(W["layer_5/weights"]), W["layer_5/bias"], relu_clip=20.0, dtype=torch.float16)
    logits = y5.double().cpu().numpy() @ w["layer_6/weights"].astype(np.float16).astype(np.float64) + w["layer_6/bias"]
    want = logits - logits.max(1, keepdims=True)
    want = (want - np.log(np.exp(want).sum(1, keepdims=True))).reshape(T, B, -1)
    got = m.acousticProbs(audio)
    for b in range(B):
        assert got[b].shape == want[:, b].shape
        assert np.abs(np.log(np.maximum(got[b], 1e-30)) - np.maximum(want[:, b], np.log(1e-30))).max() < 1e-4, b


def test_batches_streams_and_one_shot_agree(small):
    """A row's sums run in one order however many rows there are: utterances get the same bits alone, in ragged batches, in the pipelined path and, as text, fed in hops."""
    m, _ = small
    rng = np.random.RandomState(4)
    lens = (rng.uniform(0.2, 2.6, size=14) * 16000).astype(int)
    lens[3], lens[9] = 300, 0
    audio = [synth.synth_audio(int(n), seed=2300 + i) for i, n in enumerate(lens)]
    together, texts = m.acousticProbs(audio), m.sttBatch(audio)
    for i, a in enumerate(audio):
        assert np.array_equal(together[i], m.acousticProbs([a])[0]), i
        assert texts[i] == m.stt(a), i
        s = m.createStream()
        for off in range(0, len(a), 5120):
            s.feedAudioContent(a[off:off + 5120])
        assert s.finishStream() == texts[i], i
    assert any(texts)
    t = m.submitBatch(audio)
    for got, want in zip(m.batchProbs(t, len(audio)), together):
        assert np.array_equal(got, want)
    assert m.collectBatch(t) == texts


def test_chunk_carries_its_state(small):
    """STTX_InferChunk (16 rows and one): two halves with the state handed on are the whole."""
    m, _ = small
    win = np.random.RandomState(5).randn(16, 494).astype(np.float32) * 3
    z = np.zeros(256, np.float32)
    p, c, h = m.inferChunk(win, z, z)
    p1, c1, h1 = m.inferChunk(win[:7], z, z)
    p2, c2, h2 = m.inferChunk(win[7:], c1, h1)
    assert np.array_equal(np.concatenate([p1, p2]), p) and np.array_equal(c, c2) and np.array_equal(h, h2)
    assert np.allclose(p.sum(1), 1.0, atol=1e-5)


def test_wide_model_in_flight(tmp_path):
    """2048 units, pairs of batches in flight (captured recurrences, both engines' workspaces): every batch is what it is alone, the pair in either order."""
    w = synth.synth_weights(32, n_hidden=2048)
    w["layer_6/weights"] = (w["layer_6/weights"] * 6.0).astype(np.float32)
    m = _model(tmp_path, w, "wide")
    m.enableExternalScorer(os.path.join(FIX, "pruned_lm.scorer"))
    sets = [[synth.synth_audio(16000 + 800 * i, seed=700 + 64 * k + i) for i in range(24)] for k in range(3)]
    want = [m.sttBatch(s) for s in sets]
    for order in ((0, 1, 2, 0), (2, 1, 0, 1)):
        tickets = []
        for k in order:
            if len(tickets) == m.pipelineDepth():
                j, t = tickets.pop(0)
                assert m.collectBatch(t) == want[j]
            tickets.append((k, m.submitBatch(sets[k])))
        for j, t in tickets:
            assert m.collectBatch(t) == want[j]


def test_off_by_default(tmp_path):
    """A model loaded without the tunable runs in f16 beside one that has it, and the tunable changes no model that is loaded."""
    w = synth.synth_weights(33, n_hidden=128)
    a = synth.synth_audio(16000, seed=5)
    plain = _model(tmp_path, w, "a", f8=False)
    before = plain.acousticProbs([a])[0]
    f8 = _model(tmp_path, w, "b")
    native.set_tuning("am_f8", 1)
    try:
        assert plain.acousticMode() == 0 and np.array_equal(plain.acousticProbs([a])[0], before)
    finally:
        native.set_tuning("am_f8", 0)
    assert f8.acousticMode() == 2 and not np.array_equal(f8.acousticProbs([a])[0], before)


def test_wide_batches_give_an_utterance_its_own_bits(tmp_path):
    """2048 units: an utterance alone (250 rows: tiles of 32 rows, of 64 in the x half of the cell), among eight (2000 rows: 64, 256), among twenty-four (6000: 128,
    256) and among forty (10000: 256) gets the same probabilities in every bit."""
    m = _model(tmp_path, synth.synth_weights(34, n_hidden=2048), "wide2")
    audio = [synth.synth_audio(80000, seed=900 + i) for i in range(40)]
    batches = [m.acousticProbs(audio[:n]) for n in (8, 24, 40)]
    for i in (0, 3, 7, 20, 39):
        alone = m.acousticProbs([audio[i]])[0]
        assert alone.shape[0] == 250
        for among in batches:
            assert i >= len(among) or np.array_equal(alone, among[i]), (i, len(among))


@pytest.mark.parametrize("kw", [{}, {"quantize": True, "per_channel": True}, {"f16_weights": True}], ids=["f32", "int8", "f16"])
def test_any_file_takes_it(tmp_path, kw):
    """A `.tflite` export of either kind runs as the container of its (de-quantised) tensors does, also where am_i8 asks for the file's own arithmetic."""
    from stt_amd import Model, modelfile, tflitefile
    w = synth.synth_weights(35, n_hidden=256)
    p, q = str(tmp_path / "m.tflite"), str(tmp_path / "m.sttw")
    eff = tflitefile.write_tflite(p, w, synth.ENGLISH_LABELS, beam_width=64, **kw)
    modelfile.write_model(q, {n: eff[n] for n in modelfile.TENSOR_ORDER}, synth.ENGLISH_LABELS, beam_width=64)
    native.set_tuning("am_f8", 1), native.set_tuning("am_i8", 1)
    try:
        a, b = Model(p), Model(q)
    finally:
        native.set_tuning("am_f8", 0), native.set_tuning("am_i8", -1)
    assert a.acousticMode() == b.acousticMode() == 2
    audio = [synth.synth_audio(n, seed=60 + n) for n in (300, 9000, 31000)]
    for x, y in zip(a.acousticProbs(audio), b.acousticProbs(audio)):
        assert np.array_equal(x, y)
    assert a.sttBatch(audio) == b.sttBatch(audio)


def test_streams_advanced_together(small):
    """Streams that join and end at different hops, advanced by one call a hop for all of them (their passes replayed from graphs), end with what each is alone."""
    from stt_amd import model as M
    m, _ = small
    audio = [synth.synth_audio(int(n), seed=2500 + i) for i, n in enumerate((40000, 5120, 23000, 61000, 300, 17000))]
    want = [m.stt(a) for a in audio]
    assert any(want)
    for turn in range(2):
        live, got, k = [], {}, 0
        while k < len(audio) or live:
            if k < len(audio):
                live.append([k, m.createStream(), 0])
                k += 1
            M.feedAudioContentBatch([s for _, s, _ in live], [audio[i][at:at + 5120] for i, _, at in live])
            M.intermediateDecodeBatch([s for _, s, _ in live])
            for stream in live:
                stream[2] += 5120
            ended = [e for e in live if e[2] >= len(audio[e[0]])]
            if ended:
                for (i, _, _), text in zip(ended, M.finishStreamBatch([s for _, s, _ in ended])):
                    got[i] = text
                live = [e for e in live if e[2] < len(audio[e[0]])]
        assert [got[i] for i in range(len(audio))] == want, turn
