"""An id outside the vocabulary shows in the logits of its sequence, or of all sequences behind a shared prompt with it, whatever
the projections' bits."""
import pytest
import torch

from glt_b200 import decode
from test_gpu_decode_shared import HD, HID, F, L, NH, NKV, THETA, V, ids_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("bad", [-1, V, 2 ** 31 - 1])
def test_unknown_id_of_a_sequence(bits, bad):
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=4, std=0.06)
    d = decode.Decoder(w, NH, NKV, HD, seqs=3, max_tokens=40, group=32, block_tokens=16, rope_theta=THETA, bits=bits)
    ids, more = ids_of(6, 3, 9), ids_of(7, 3, 1)
    want = [d.step(ids), d.step(more)]
    assert all(torch.isfinite(y).all() for y in want)
    d.reset()
    wrong = ids.clone()
    wrong[1, 3] = bad
    for x, y in zip((wrong, more), want):   # the cache holds its tokens from then on
        got = d.step(x)
        assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2]], y[[0, 2]])
    d.reset()
    logps = d.generate(wrong, 3)[1]
    assert torch.isnan(logps[1]).all() and torch.isfinite(logps[[0, 2]]).all()
    d.reset()
    assert torch.equal(d.step(ids), want[0])


def test_all_sequences_unknown():
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=4, std=0.06)
    d = decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=40, rope_theta=THETA)
    assert torch.isnan(d.step(torch.full((2, 1), V, device="cuda", dtype=torch.int64))).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [-1, V, 2 ** 31 - 1])
def test_unknown_id_in_a_shared_prompt(bits, fmt, bad):
    w = decode.random_weights(HID, F, L, NH, NKV, HD, V, seed=4, std=0.06)
    d = decode.Decoder(w, NH, NKV, HD, seqs=2, max_tokens=40, group=32, block_tokens=16, fmt=fmt, rope_theta=THETA, bits=bits,
                       shared_tokens=70)
    prompt, ids = ids_of(5, 50), ids_of(6, 2, 9)
    d.share(prompt)
    want = d.step(ids)
    assert torch.isfinite(want).all()
    d.reset()
    wrong = prompt.clone()
    wrong[17] = bad
    d.share(wrong)
    assert torch.isnan(d.step(ids)).all() and torch.isnan(d.step(ids[:, :1])).all()
    d.reset()
    assert torch.isnan(d.generate(ids, 3)[1]).all()
    d.reset()   # the prompt stays, and so does its mark
    assert torch.isnan(d.step(ids)).all()
    d.reset()
    d.share(prompt)
    assert torch.equal(d.step(ids), want)
