"""What the decoding example refuses on the host, before any launch (no GPU: nothing of the model is built)."""
import sys

import pytest
import torch

from glt_b200 import decode


@pytest.fixture
def decoder(monkeypatch):
    """A decoder for 2 sequences of up to 10 tokens whose steps only note how many tokens they bring."""
    d = decode.Decoder.__new__(decode.Decoder)
    d.seqs, d.max_tokens, d.held, d.steps = 2, 10, 0, []
    d.embed = torch.zeros(4, 64)
    d.lengths = torch.zeros(2, dtype=torch.int32)

    def step(ids):
        d.steps.append(ids.shape[1])
        return torch.zeros(2, 4)

    class Top:
        top_ids, top_logp = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1)

    monkeypatch.setattr(d, "_step", step)
    monkeypatch.setattr(decode.serve, "token_logprobs", lambda *a, **k: Top)
    monkeypatch.setattr(torch.cuda, "device", lambda index: torch.no_grad())
    return d


def ids(n, seqs=2, dtype=torch.int32):
    return torch.zeros(seqs, n, dtype=dtype)


def test_steps_past_the_cache_are_refused(decoder):
    """One token too many would index the rotary table past its end."""
    decoder.step(ids(9))
    with pytest.raises(ValueError, match="max_tokens"):
        decoder.step(ids(2))
    decoder.step(ids(1))
    with pytest.raises(ValueError, match="max_tokens"):
        decoder.step(ids(1))
    assert decoder.steps == [9, 1] and decoder.held == 10
    decoder.reset()
    decoder.step(ids(10))
    assert decoder.held == 10


def test_generations_past_the_cache_are_refused_before_their_prompt(decoder):
    with pytest.raises(ValueError, match="max_tokens"):
        decoder.generate(ids(7), 5)          # the last token is not fed back: 7 + 4
    assert decoder.steps == [] and decoder.held == 0
    decoder.generate(ids(7), 4)
    assert decoder.steps == [7, 1, 1, 1] and decoder.held == 10


@pytest.mark.parametrize("bad", [ids(0), ids(3, seqs=1), ids(3, seqs=3), torch.zeros(2, dtype=torch.int32),
                                 ids(3, dtype=torch.float32)])
def test_ids_of_another_shape_or_type_are_refused(decoder, bad):
    with pytest.raises(ValueError, match="ids"):
        decoder.step(bad)
    assert decoder.steps == []


@pytest.mark.parametrize("tokens", [0, -1])
def test_no_tokens_to_generate_are_refused(decoder, tokens):
    with pytest.raises(ValueError, match="tokens"):
        decoder.generate(ids(3), tokens)
    assert decoder.steps == []


@pytest.mark.parametrize("args", [["--tokens", "0"], ["--prompt", "0"], ["--seqs", "0"]])
def test_the_command_refuses_empty_work(monkeypatch, args):
    monkeypatch.setattr(sys, "argv", ["decode"] + args)
    monkeypatch.setattr(decode, "random_weights", lambda **k: pytest.fail("weights were made"))
    with pytest.raises(SystemExit):
        decode.main()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_ids_outside_the_vocabulary_give_their_sequence_nan(dtype):
    """An index out of range would end the context, and a negative one would silently count from the end."""
    d = decode.Decoder.__new__(decode.Decoder)
    d.embed = torch.randn(7, 64).to(torch.bfloat16)
    good = torch.tensor([[0, 6, 3]], dtype=dtype)
    for bad in (7, -1, 2 ** 31 - 1, -2 ** 31):
        x = d._lookup(torch.cat((good, torch.tensor([[5, bad, 2]], dtype=dtype), good)))
        assert torch.equal(x[:3], d.embed[[0, 6, 3]]) and torch.equal(x[6:], x[:3])
        assert torch.isnan(x[3:6]).all() and x.dtype == torch.bfloat16
