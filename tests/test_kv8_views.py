"""What layers hand on of their cache's view (no GPU)."""

from types import SimpleNamespace

import torch

from llm_pipeline_b200.cache import KVPagesSpec, StateSpec
from llm_pipeline_b200.parts.base import LayerCache
from llm_pipeline_b200.parts.side_by_side import SideBySide


class Seen:
    """A mixer that keeps the view it is given."""

    w_in = None

    def cache_spec(self):
        return KVPagesSpec(2, 16)

    def forward(self, x, ctx, cache):
        self.cache = cache
        return torch.zeros(1, 4), None

    forward_deferred = forward


VIEW = dict(pages=torch.zeros(3, 128, dtype=torch.uint8), group=1, state=torch.arange(12.0).view(2, 6), writes=False, page_size=8)


def same_but_state(view):
    assert view.pages.data_ptr() == VIEW["pages"].data_ptr() and (view.group, view.writes, view.page_size) == (1, False, 8)


def test_a_mixer_behind_an_input_convolution_sees_the_whole_view():
    from llm_pipeline_b200.parts.block import ParallelResidualBlock as Block

    block, mixer = object.__new__(Block), Seen()
    block._own_state, block._mixer_state, block.mixer, block.feed_forward = 2, StateSpec((4,), torch.float32), mixer, None
    block._inputs = lambda stream, ctx, cache: (torch.zeros(1, 4), torch.zeros(1, 4))
    block.forward(SimpleNamespace(add=lambda *a: None), None, LayerCache(**VIEW))
    same_but_state(mixer.cache)
    assert torch.equal(mixer.cache.state, VIEW["state"][:, 2:])


def test_mixers_side_by_side_see_the_whole_view():
    both = object.__new__(SideBySide)
    both.members, both._state_at, both.w_in = [Seen(), Seen()], [(0, 2), (2, 6)], None
    both._results(torch.zeros(1, 4), None, LayerCache(**VIEW))
    for m, (a, b) in zip(both.members, both._state_at):
        same_but_state(m.cache)
        assert torch.equal(m.cache.state, VIEW["state"][:, a:b])
