"""Orderings between the lanes of a warp that the serving kernels rely on
(CPU only): a store of one lane and a load of another are ordered by
__syncwarp or __syncthreads alone; shuffles, votes and reductions order no
memory, and no run on a GPU shows their absence."""

import os

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grokking_abmod_b200", "csrc")


def _between(name, kernel, start, end):
    """The text of a kernel between two of its statements."""
    text = open(os.path.join(CSRC, name)).read()
    text = text[text.index("\n    " + kernel + "("):]
    text = text[text.index(start) + len(start):]
    return text[:text.index(end)]


def test_scales_of_the_first_tiles_are_ordered_before_their_reads():
    """Lane 0 writes a tile's scales behind its copies; every lane reads them
    after the copies' barrier, which the write comes after."""
    prologue = _between("cache_attention.cu", "attend_split", "issue(issued);", "const float4 sc = meta[s];")
    assert "__syncwarp();" in prologue[:prologue.index("for (int n = 0; n < mine; ++n)")]
    loop = _between("cache_attention.cu", "attend_split", "for (int n = 0; n < mine; ++n)", "// The four warps' results")
    assert loop.rindex("__syncwarp();") > loop.rindex("load_words<VW>")


def test_scales_are_read_by_every_lane_before_one_writes_them():
    """A page's earlier scales are read by the whole group; its first thread
    stores the new ones."""
    text = _between("cache_ops.cu", "write_pages", "before[1] = *scale_at[1];", "*scale_at[which] = scale")
    wide, narrow = text.index("if constexpr (G > 32)"), text.index("} else {\n    __syncwarp();")
    assert wide < text.index("__syncthreads();") < narrow


def test_a_copy_whose_wait_ran_out_is_waited_for_again():
    """With the ones behind it: none may land when the block has ended."""
    text = _between("cache_attention.cu", "attend_split", "*gave_up = 1;", "break;")
    assert "for (int k = n; k < issued; ++k) tc::bar_wait(" in text
