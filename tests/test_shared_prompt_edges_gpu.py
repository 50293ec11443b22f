"""channel_b200.shared_prompt: what decode refuses, and its logits against a plain decoder."""
import pytest
import torch

from channel_b200 import _lib as L
from channel_b200.shared_prompt import DecoderShape, SharedPromptDecoder


@pytest.mark.parametrize("prompt,streams,n", [([], 2, 3), ([1, 2], 0, 3), ([1, 2], 2, 0), ([1, 2], 2, -1), ([1, -1], 2, 3),
                                              ([4096], 2, 3), ([5, 1 << 40], 2, 3)])
def test_decode_refuses(prompt, streams, n):
    decoder = SharedPromptDecoder.__new__(SharedPromptDecoder)  # the checks come before any work
    decoder.shape = DecoderShape()
    with pytest.raises(L.ChannelError):
        decoder.decode(prompt, streams, n)
