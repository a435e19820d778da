"""The block-128 product's slots for TMA stores: a slot in shared memory is written again only when the store that last read it is
done.  A warp that overwrites one too early gives wrong columns without any error, so the protocol is read from the source and followed
here, over sequences of tiles whose last columns lie beyond N; the kernel itself runs such tiles in test_block_epilogue_gpu.py."""

import itertools
import re

from test_kernel_waits_cpu import _functions


def _protocol():
    """(whether a piece beyond N commits a group, the groups that may be pending when a slot is written), as text of the source."""
    body = next(b for h, b in _functions("block_gemm.cu") if "block_gemm_kernel(" in h)
    loop = re.search(r"for \(int c = 0; c < C::kCols; c \+= 32\) \{\s*const int col = t\.n0 \+ part \* C::kCols \+ c;\s*if \(col >= p\.n\) (.*?)"
                     r"const uint32_t slot = (.*?);.*?bulk_wait_read<(.*?)>\(\).*?tma_store_2d.*?bulk_commit\(\);", body, re.S)
    skipped, slot, pending = loop.groups()
    assert slot == "slots + c / 32 % C::kEpiSlots * 2048" and pending == "C::kEpiSlots - 1"
    assert "break" in skipped or "continue" in skipped
    return "bulk_commit()" in skipped and "continue" in skipped


def _first_overwrite(commits, pieces, slots, tiles):
    """The first (tile, piece) that writes a slot whose last store may still be reading; None if there is none.  ``tiles``: the
    pieces of each that lie inside of N, the others follow them."""
    groups = []  # slot that each committed group reads, None for an empty one
    for i, inside in enumerate(tiles):
        for piece in range(pieces):
            if piece >= inside:
                if commits:
                    groups.append(None)
                    continue
                break
            slot = piece % slots
            if slot in groups[len(groups) - (slots - 1):]:  # all before are done
                return i, piece
            groups.append(slot)
    return None


def test_a_slot_is_written_when_its_last_store_is_done():
    commits = _protocol()
    for pieces, slots in ((1, 1), (2, 1), (2, 2), (4, 4)):  # columns of a warp / 32, slots: 64, 128, 192 and 256 columns
        for tiles in itertools.product(range(pieces + 1), repeat=4):
            assert _first_overwrite(commits, pieces, slots, tiles) is None, (pieces, slots, tiles)


def test_the_protocol_check_sees_a_warp_that_leaves_early():
    assert _first_overwrite(False, 2, 2, (1, 2)) == (1, 0)
    assert _first_overwrite(False, 4, 4, (3, 1)) == (1, 0)
    assert _first_overwrite(False, 2, 1, (1, 2, 0, 1)) is None


def test_slots_and_columns_are_those_of_the_configuration():
    with open(__file__.replace("tests/test_block_epilogue_cpu.py", "halops_b200/csrc/block_gemm.cu")) as f:
        text = f.read()
    assert "kEpiSlots = kRowScales ? 0 : BN == 256 ? 4 : BN == 192 ? 2 : 1;" in text
    assert "kParts = BN == 192 ? 3 : 2;" in text and "kCols = BN / kParts;" in text
