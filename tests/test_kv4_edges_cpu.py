"""The paged cache held in 4 bits without a GPU, where it can go wrong: the order of hand-offs in its sources."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "ssd_b200" / "csrc"


def _source(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


# ---------------------------------------------------------------------------------------------------- order
def test_positions_are_written_before_their_chunk_is_announced():
    """Four lanes of the copying warp write where a chunk's keys are, one lane arrives for all of them: a vote orders no memory, so a barrier of the warp stands between them."""
    body = _source("kv4_tiles.cuh")
    written = [m.end() for m in re.finditer(r"codes_pos\[c\]\[lane\]\s*=", body)]
    arrives = [m.start() for m in re.finditer(r"mbar_arrive_expect_tx\(&codes_full", body)]
    assert len(written) == len(arrives) == 1
    between = body[written[0]:arrives[0]]
    assert "__syncwarp()" in between and between.rindex("__syncwarp()") < between.rindex("if (lane == 0)")
