"""The serving operators together (channel_b200.shared_prompt): streams that share a prompt's
pages decode what streams with copies of their own decode."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decoder(ctx):
    from channel_b200.shared_prompt import DecoderShape, SharedPromptDecoder
    return SharedPromptDecoder(ctx, DecoderShape(), 600)


PROMPT = [(37 * i + 11) % 4096 for i in range(45)]


def test_shared_pages_give_the_tokens_of_own_copies(decoder):
    shared = decoder.decode(PROMPT, 20, 12)
    own = decoder.decode(PROMPT, 20, 12, share=False)
    assert torch.equal(shared, own)
    assert bool((shared == shared[0]).all())  # one prompt, greedy: every stream alike
    assert len(set(shared[0].tolist())) > 1


def test_streams_sample_their_own_continuations(decoder):
    a = decoder.decode(PROMPT, 24, 10, temperature=1.0, top_k=50, top_p=0.95)
    b = decoder.decode(PROMPT, 24, 10, temperature=1.0, top_k=50, top_p=0.95)
    c = decoder.decode(PROMPT, 24, 10, temperature=1.0, top_k=50, top_p=0.95, seed=2)
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert len({tuple(r) for r in a.tolist()}) > 12
    assert int(a.min()) >= 0 and int(a.max()) < 4096


def test_top_k_of_one_is_greedy(decoder):
    assert torch.equal(decoder.decode(PROMPT, 3, 6, temperature=1.0, top_k=1), decoder.decode(PROMPT, 3, 6))
