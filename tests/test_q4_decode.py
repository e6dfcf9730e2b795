"""The attention block over the 4-bit cache (kernelfoundry_b200.q4_decode) without a GPU: slots and room."""
from __future__ import annotations

import pytest
import torch


def _block(**kw):
    from kernelfoundry_b200.q4_decode import Q4AttentionBlock

    return Q4AttentionBlock(3, 100, 64, 2, 1, 64, 16, device="cpu", **kw)      # 7 pages of 16 tokens a sequence


def test_slots_of_tokens_padding_and_positions_past_the_table():
    """Padding of a chunk may end past the table: it has no slot, like padding inside it; tokens have theirs."""
    block = _block()
    positions = (60 + torch.arange(64)).expand(3, 64)                          # pages 3 to 7, of which 7 does not exist
    lens = torch.tensor([40, 1, 17])
    valid = torch.arange(64) < lens[:, None]
    got = block.slots(positions, valid)
    assert got.dtype == torch.int32 and got.shape == (3, 64)
    for b in range(3):
        for i in range(64):
            p = 60 + i
            want = int(block.table[b, p // 16]) * 16 + p % 16 if i < lens[b] else -1
            assert int(got[b, i]) == want
    all_ = block.slots(positions)
    assert (all_[:, 52:] == -1).all() and (all_[:, :52] >= 0).all()            # 112 tokens have room
    assert (block.slots(torch.full((3, 1), 1 << 40)) == -1).all()


def test_prefill_refuses_what_does_not_fit():
    block = _block()
    assert block.capacity == 112
    for S, past, lens in ((113, 0, None), (64, 60, None), (64, 60, [53, 1, 1]), (64, 100, [13, 1, 1]), (8, 120, None)):
        with pytest.raises(ValueError, match="room for 112"):
            block.prefill(torch.zeros(3, S, 64).half(), None if lens is None else torch.tensor(lens, dtype=torch.int32), past=past)


def test_step_refuses_what_does_not_fit():
    block = _block()
    for lens, S in (([112, 0, 5], 1), ([3, 111, 5], 2), ([0, 0, 110], 3)):
        block.lens.copy_(torch.tensor(lens))
        block._most = 112                                                      # an upper bound; the lengths decide
        with pytest.raises(ValueError, match="room for 112"):
            block.step(torch.zeros(3, S, 64).half())
        assert block.lens.tolist() == lens


def test_steps_after_a_capture_look_at_the_lengths():
    """Replays move the lengths unseen: the host's own count says nothing any more."""
    block = _block()
    block._captured = True
    block.lens.copy_(torch.tensor([112, 0, 0]))
    with pytest.raises(ValueError, match="room for 112"):
        block.step(torch.zeros(3, 1, 64).half())


@pytest.mark.parametrize("args", [("--steps", "0"), ("--prompt", "1"), ("--batch", "0")])
def test_command_refuses_empty_runs(args, capsys):
    from kernelfoundry_b200.q4_decode import main

    with pytest.raises(SystemExit):
        main(list(args))
    assert "at least" in capsys.readouterr().err
