"""The graphs that decoding on the GPU keeps."""

import pytest

import util
from test_device_decode_gpu import begin, folders, make  # noqa: F401

pytestmark = pytest.mark.gpu


def test_only_the_last_graphs_are_kept(folders, monkeypatch):  # noqa: F811
    """More batch sizes than there is room for: the one that was used longest ago goes, and comes back with the same tokens."""
    from oxr_inference_b200.engine import device_decode

    monkeypatch.setattr(device_decode, "LOOPS", 2)
    prompts = [util.token_ids("A", n, seed=70 + n) for n in (9, 14, 21)]

    def decoded(sizes):
        r = make(folders["A"], "A", "float32", "e4m3")
        caches, tokens = begin(r, prompts)
        out, kept = [list(t) for t in zip(tokens)], []
        for n in sizes:
            for o, more in zip(out, r.decode(caches[:n], [o[-1] for o in out[:n]], 3)):
                o += more
            kept.append([k[0] for k in r._device_decode._loops])
        r.cache.check()
        return out, kept

    out, kept = decoded((3, 2, 3, 1, 2, 3, 3))
    assert kept == [[3], [3, 2], [2, 3], [3, 1], [1, 2], [2, 3], [2, 3]]
    monkeypatch.setattr(device_decode, "LOOPS", 8)
    assert decoded((3, 2, 3, 1, 2, 3, 3))[0] == out


def test_tokens_outside_the_vocabulary_are_refused_before_anything_moves(tmp_path):
    """Recurrent states cannot be taken back once a step has run."""
    import radapel_util

    folder = radapel_util.make_folder(tmp_path, radapel_util.MODEL_X, "x", 3)
    r, s = (make(folder, "radapel", "float32", page=8) for _ in range(2))
    prompts = [[5, 17, 3, 9], [9, 8, 7]]
    (caches, tokens), (caches2, tokens2) = begin(r, prompts), begin(s, prompts)
    free = s.cache.free_pages
    for bad in (-1, s.model.spec.vocab_size, 1 << 40):
        with pytest.raises(ValueError, match="vocabulary"):
            s.decode(caches2, [tokens2[0], bad], 4)
    assert s.cache.free_pages == free and [rc.length for rc in caches2] == [4, 3]
    assert s.decode(caches2, tokens2, 4) == r.decode(caches, tokens, 4)
