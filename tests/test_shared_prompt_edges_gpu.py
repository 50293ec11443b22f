"""channel_b200.shared_prompt: what decode refuses, and its logits against a plain decoder."""
import pytest
import torch

from channel_b200 import _lib as L
from channel_b200.paged import plan_pages
from channel_b200.shared_prompt import DecoderShape, SharedPromptDecoder


@pytest.mark.parametrize("prompt,streams,n", [([], 2, 3), ([1, 2], 0, 3), ([1, 2], 2, 0), ([1, 2], 2, -1), ([1, -1], 2, 3),
                                              ([4096], 2, 3), ([5, 1 << 40], 2, 3)])
def test_decode_refuses(prompt, streams, n):
    decoder = SharedPromptDecoder.__new__(SharedPromptDecoder)  # the checks come before any work
    decoder.shape = DecoderShape()
    with pytest.raises(L.ChannelError):
        decoder.decode(prompt, streams, n)


@pytest.fixture(scope="module")
def decoder(ctx):
    return SharedPromptDecoder(ctx, DecoderShape(), 64)


def start(streams, columns=2):
    """no tokens yet, and free pages"""
    return (torch.zeros(streams, dtype=torch.int32, device="cuda"),
            torch.full((streams, columns), -1, dtype=torch.int32, device="cuda"),
            torch.arange(20, 60, dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
def test_a_step_from_another_stream(decoder):
    """tokens and plan come from work on the caller's stream that takes a while, and the logits are
    read there"""
    lens, table, free = start(5)
    ids = torch.tensor([3, 9, 27, 81, 243], device="cuda")
    big = torch.randn(8192, 8192, device="cuda")

    def one():
        late = (big @ big @ big).abs().sum().clamp(max=0).long()  # 0
        plan = plan_pages(lens, torch.ones_like(lens) + late.int(), table, free, 16, 5)
        logits = decoder.step(ids + late, plan)
        return logits.clone()
    with torch.cuda.stream(decoder.stream):
        ref = one()
    decoder.stream.synchronize()
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        decoder.k_pool.zero_(), decoder.v_pool.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            got = one()
        stream.synchronize()
        assert torch.equal(got, ref)
    assert torch.isfinite(ref).all() and int(decoder.status.item()) == 0


@pytest.mark.gpu
def test_rows_of_nan_are_not_tokens(decoder):
    """an activation that is not a number ends in an error, not in token -1"""
    with torch.cuda.stream(decoder.stream):
        row = decoder.embed[7].clone()
        decoder.embed[7] = float("nan")
    try:
        for share in (True, False):
            with pytest.raises(L.ChannelError, match="nothing to choose"):
                decoder.decode([1, 7], 3, 2, share=share)
    finally:
        with torch.cuda.stream(decoder.stream):
            decoder.embed[7] = row
    assert int(decoder.decode([1, 8], 3, 2).min()) >= 0
