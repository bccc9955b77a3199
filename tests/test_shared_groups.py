"""What the launches with shared prefixes rest on, as read from their source."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "attention_kernel_triton_amd" / "csrc"


def test_the_groups_places_are_stored_before_other_lanes_look_at_them():
    """One wave rewrites the groups' places in LDS and then finds the lengths from them, an entry by
    another lane than the one that stored it: the two are ordered."""
    text = (CSRC / "paged_chunk.hip").read_text()
    kernel = text[text.index("void paged_chunk_kernel(ChunkParams p)"):]
    stored = kernel.rindex("sm_table[b] = int4{q0")
    read = kernel.index("shared_shares<D>(p, table, W)", stored)
    assert re.search(r"wave_lds_sync\(\)|__syncthreads\(\)", kernel[stored:read])
