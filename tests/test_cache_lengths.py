"""What a dense layer says of its rows after cuts (CPU)."""

from __future__ import annotations

import copy
import pickle
import random

import torch


def test_least_since_is_the_fewest_tokens_left() -> None:
    """Random growth and cuts, against a record of every cut; also through copies of the layer, which go on by themselves."""
    from lazykv_amd.cache import DenseLayer

    rng = random.Random(1)
    for through in (lambda x: x, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        layer, kv = DenseLayer(64), torch.zeros((1, 1, 1, 4))
        layer.store(kv, kv)
        marks: list[list[int]] = []  # (cuts then, fewest tokens left since)
        for step in range(400):
            if step % 100 == 50:
                layer = through(layer)
            if rng.random() < 0.6 and layer.length < 64:
                n = rng.randint(1, 64 - layer.length)
                layer.store(kv.expand(1, 1, n, 4), kv.expand(1, 1, n, 4))
            else:
                cut = rng.randint(0, layer.length) if rng.random() < 0.7 else layer.length
                layer.reset() if cut == 0 else layer.truncate(cut)
                marks = [[c, min(least, cut)] for c, least in marks]
            if rng.random() < 0.3:
                marks.append([layer.cuts, 65])
            for cuts, least in marks[-20:]:
                assert layer.least_since(cuts) == (least if least < 65 else layer.length)
