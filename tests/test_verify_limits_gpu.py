"""Verifying drafted tokens through the engine where room is short: memory for graphs, nodes of a step, windows, pieces of which one fails; latents that
serve as keys and values."""
import random

import pytest
import torch

from test_trees_gpu import TOL, folders, path_to, random_tree, rel_err, vocab_of        # noqa: F401 (folders is a fixture)
from tiny_models import _dense, _latent, _layer, prompt, write_pipilix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("windows", [(50, 7), (9, 50), (None, 12)])
def test_layers_that_read_anothers_cache_through_another_window(tmp_path, windows):
    """Drafts down to the narrowest window change no answer (32-bit); deeper ones are refused."""
    from rocml_b200 import Engine, RocmlError, StepEntry, TreeEntry
    from tiny_models import _KA_ROT, _kdiff, write_kemizen
    config = {"architecture": "Kemizen", "vocab": 211, "width": 64, "embedding": {"scale": 1.5}, "norm": {"eps": 1e-6},
              "layers": [_kdiff(4, 2, 12, 20, 0.5, 0.3, _KA_ROT, 96, size=windows[0], softcap=3.0),
                         _kdiff(4, 2, 12, 20, 0.7, 0.5, _KA_ROT, 48, size=windows[1], softcap=5.0, kv_from=0)]}
    write_kemizen(str(tmp_path), config, seed=4)
    eng = Engine.from_folder(str(tmp_path), dtype="float32", max_tokens=1024, max_slots=3)
    deepest = min(w for w in windows if w)
    ids, way = prompt(5, 70, 211), prompt(6, deepest, 211)
    slot = eng.new_sequence()
    eng.step([StepEntry(slot, ids)])
    got = eng.tree_logits([TreeEntry(slot, way + [3, 4], list(range(-1, deepest - 1)) + [0, 1])]).clone()
    paths = [way[:i + 1] for i in range(deepest)] + [way[:1] + [3], way[:2] + [4]]
    for g, path in zip(got, paths):
        other = eng.new_sequence()
        want = eng.step([StepEntry(other, ids + path, [70 + len(path) - 1])])
        eng.release(other)
        assert rel_err(g[None], want) < 2 * TOL["float32"]
    with pytest.raises(RocmlError, match="window"):
        eng.tree_logits([TreeEntry(slot, way + [1], list(range(-1, deepest)))])
