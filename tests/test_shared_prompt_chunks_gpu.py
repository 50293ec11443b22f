"""channel_b200.shared_prompt with several tokens a step: prompts in chunks, scores of texts, and
decoding with drafts, around the operators that serve them."""
import pytest
import torch

from channel_b200 import ChannelError
from channel_b200.paged import plan_pages
from channel_b200.shared_prompt import DecoderShape, SharedPromptDecoder
from tests.gpu_util import rel_err
from tests.test_shared_prompt_edges_gpu import PlainDecoder, start

PROMPT = [(37 * i + 11) % 4096 for i in range(45)]


@pytest.mark.parametrize("call", [
    lambda d: d.decode([1, 2], 2, 3, chunk=-1), lambda d: d.score([]), lambda d: d.score([[1]]), lambda d: d.score([[1, 4096]]),
    lambda d: d.score([[1, 2]], chunk=0), lambda d: d.decode_drafted([], 1, 1), lambda d: d.decode_drafted([1, -1], 1, 1),
    lambda d: d.decode_drafted([1], 0, 1), lambda d: d.decode_drafted([1], 1, 0), lambda d: d.decode_drafted([1], 1, 1, depth=-1),
    lambda d: d.decode_drafted([1], 1, 1, branches=-1)])
def test_refused(call):
    decoder = SharedPromptDecoder.__new__(SharedPromptDecoder)  # the checks come before any work
    decoder.shape = DecoderShape()
    with pytest.raises(ChannelError):
        call(decoder)


def test_drafts_share_what_begins_alike():
    tokens, parents, depths = SharedPromptDecoder._draft([5, 1, 2, 3, 5, 1, 2, 9, 5], 3, 2)
    assert tokens == [5, 1, 2, 9, 3] and parents == [-1, 0, 1, 2, 2] and depths == [0, 1, 2, 3, 3]
    assert SharedPromptDecoder._draft([1, 2, 3], 3, 2) == ([3], [-1], [0])


@pytest.mark.parametrize("depth,branches", [(5000, 2), (3000, 3), (4095, 1), (4096, 1)])
def test_drafts_are_no_larger_than_a_tree_may_be(depth, branches):
    body = [9] + list(range(10, 4010))
    text = sum((body + [4000 + j, *range(10, 3000), j] for j in range(3)), []) + [9]
    tokens, parents, depths = SharedPromptDecoder._draft(text, depth, branches)
    assert 1 + min(depth, 4095) <= len(tokens) == len(parents) == len(depths) <= 4096
    assert parents[0] == -1 and all(0 <= p < i and depths[i] == depths[p] + 1 for i, p in enumerate(parents) if i)


@pytest.fixture(scope="module")
def decoder(ctx):
    return SharedPromptDecoder(ctx, DecoderShape(), 600)


@pytest.mark.gpu
def test_chunks_against_a_plain_decoder(decoder, oracle):
    """Logits of every token of ragged chunks, alone and behind a shared prompt (the bound of
    test_steps_against_a_plain_decoder: weights and outputs rounded to f16, as there)."""
    s, prompt = decoder.shape, [(37 * i + 11) % 4096 for i in range(21)]
    with torch.cuda.stream(decoder.stream):
        plain = PlainDecoder(oracle, s, decoder.embed.cpu().numpy())
        lens, table, free = start(1, 3)
        for chunk in (prompt[:1], prompt[1:18], prompt[18:]):
            plan = plan_pages(lens, torch.full_like(lens, len(chunk)), table, free, 16, len(chunk))
            free = free[int(plan.counts[1]):]
            logits = decoder.extend(torch.tensor(chunk, device="cuda"), plan, lens).cpu().numpy()
            lens = plan.lens
            for row, token in zip(logits, chunk):
                assert rel_err(row, plain.step(token)) < 1e-2
        streams = [plain.fork() for _ in range(3)]
        shared = table[0, :2].contiguous()
        lens, table, _ = start(3, 3)
        for sizes in ((3, 0, 17), (1, 5, 2)):
            chunks = [[(911 * b + 77 * i + 5) % 4096 for i in range(n)] for b, n in enumerate(sizes)]
            plan = plan_pages(lens, torch.tensor(sizes, dtype=torch.int32, device="cuda"), table, free, 16, sum(sizes), len(prompt))
            free = free[int(plan.counts[1]):]
            logits = decoder.extend(torch.tensor(sum(chunks, []), device="cuda"), plan, lens, shared, len(prompt)).cpu().numpy()
            lens = plan.lens
            for row, (b, token) in zip(logits, ((b, x) for b, c in enumerate(chunks) for x in c)):
                assert rel_err(row, streams[b].step(token)) < 1e-2
    assert int(decoder.status.item()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 7, 16, 64])
@pytest.mark.parametrize("share", [True, False])
def test_prompts_in_chunks_give_likely_tokens(decoder, chunk, share):
    """Greedy tokens behind a prompt in chunks: each is the likeliest by the decoder's own scores, or
    as likely but for the roundings in which the two ways differ."""
    tokens = decoder.decode(PROMPT, 3, 8, chunk=chunk, share=share)
    assert bool((tokens == tokens[0]).all())
    r = decoder.score([PROMPT + tokens[0].tolist()], top=1)[0]
    short = r.top_logprobs[-8:, 0] - r.logprobs[-8:]
    assert float(short.max()) < 0.05 and int(r.ranks[-8:].max()) <= 3


@pytest.mark.gpu
def test_scores_of_texts(decoder):
    """Texts of different lengths together and alone, in chunks of different sizes, say the same."""
    texts = [[(37 * i + 11 * b) % 4096 for i in range(n)] for b, n in enumerate((2, 50, 17, 33))]
    together = decoder.score(texts, top=3, chunk=16)
    for text, r in zip(texts, together):
        assert r.logprobs.shape == (len(text) - 1,) and r.top_ids.shape == (len(text) - 1, 3)
        alone = decoder.score([text], top=3, chunk=64)[0]
        assert float((alone.logprobs - r.logprobs).abs().max()) < 0.05
        assert float((alone.entropy - r.entropy).abs().max()) < 0.05
        assert bool((r.logprobs <= r.top_logprobs[:, 0]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("depth,branches", [(0, 0), (3, 1), (4, 2), (8, 3)])
def test_drafted_tokens_are_likely(decoder, depth, branches):
    """Greedy decoding with drafts of a text that repeats itself: every token is the likeliest after
    what is in front of it, whether it was drafted or not."""
    prompt = (PROMPT[:9] * 5)[:40]
    texts = decoder.decode_drafted(prompt, 4, 30, depth=depth, branches=branches)
    assert [len(x) for x in texts] == [30] * 4 and all(x == texts[0] for x in texts)
    r = decoder.score([prompt + texts[0]], top=1)[0]
    assert float((r.top_logprobs[-30:, 0] - r.logprobs[-30:]).max()) < 0.05 and int(r.ranks[-30:].max()) <= 3


@pytest.mark.gpu
def test_drafted_streams_sample_their_own_continuations(decoder):
    prompt = (PROMPT[:9] * 5)[:40]
    a = decoder.decode_drafted(prompt, 12, 20, temperature=1.0, top_k=50)
    b = decoder.decode_drafted(prompt, 12, 20, temperature=1.0, top_k=50)
    c = decoder.decode_drafted(prompt, 12, 20, temperature=1.0, top_k=50, seed=2)
    assert a == b and a != c and len({tuple(x) for x in a}) > 6


@pytest.mark.gpu
def test_drafts_are_accepted(decoder):
    """A step's tree behind a cache: with the tokens that greedy decoding takes as drafts, all are kept."""
    text = decoder.decode_drafted(PROMPT, 1, 6, depth=0)[0]
    calls = []
    real = SharedPromptDecoder._draft
    try:
        # the tree is the rest of the known text, beside a wrong branch
        def known(seen, depth, branches):
            done = len(seen) - len(PROMPT)
            rest = text[done:]
            calls.append(done)
            return [seen[-1], 4095] + rest, [-1, 0] + [0] + list(range(2, 1 + len(rest))) if rest else [-1, 0], \
                [0, 1] + list(range(1, 1 + len(rest)))
        SharedPromptDecoder._draft = staticmethod(known)
        assert decoder.decode_drafted(PROMPT, 1, 6)[0] == text
    finally:
        SharedPromptDecoder._draft = real
    assert calls == [1]  # one step for the five tokens after the first


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["score", "decode"])
def test_results_outlive_the_next_call(decoder, what):
    """Results read by work that is still queued on the caller's stream when they are let go of and
    the decoder is called again."""
    def call(seed):
        texts = [[(seed * 31 + 7 * b + 13 * i) % 4096 for i in range(40)] for b in range(6)]
        if what == "score":
            return [t for r in decoder.score(texts, top=3) for t in r]
        return [decoder.decode(texts[0], 6, 24, chunk=40, temperature=1.0, seed=seed)]

    want = [t.clone() for t in call(1)]
    call(2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(400_000_000)  # 0.2 s: longer than the next calls
            results = call(1)
            got = [t.clone() for t in results]
            del results
            call(2)
            call(3)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
