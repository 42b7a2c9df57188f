"""What captured decode steps read stays theirs when the model's weights change."""
import weakref

import pytest
import torch

from graphs import DecodeGraphs
from test_q8_model_gpu import CFG, cache_for, make, tokens

pytestmark = pytest.mark.gpu


def test_transposed_copies_live_as_long_as_the_graph():
    """A step of 20 rows multiplies by a transposed copy of the head's weight.  A changed weight replaces the copy on the
    next such step; the one that the graph reads is not freed for it."""
    model, cache = make(), cache_for(blocks=256)
    graphs = DecodeGraphs(model, cache, buckets=(20,))
    copy = weakref.ref(model.embed_tokens.weight._mi_transposed[1])
    with torch.no_grad():
        model.embed_tokens.weight[3] *= 2
    g = torch.Generator().manual_seed(1)
    model(tokens(g, 20, 1), cache, [cache.alloc() for _ in range(20)])
    assert model.embed_tokens.weight._mi_transposed[1] is not copy()
    assert copy() is not None and copy().shape == (CFG.hidden_size, CFG.vocab_size)
    assert graphs.run([cache.alloc()], [5]).shape == (1, CFG.vocab_size)
