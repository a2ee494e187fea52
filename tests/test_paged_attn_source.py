"""The order of a flag in LDS, read off the source (no GPU needed): the attention kernel over pages has forms whose waves meet no
barrier in a unit's stages, so a wave that is ahead may set `odd` for the next unit while a late one is still in the last."""
import os
import re

from conftest import PKG


def test_the_flag_of_left_out_values_is_read_in_one_place():
    """Every read of `odd` stands between the barrier that ends a unit's stages and the next barrier; barriers further down hold
    the fast waves up until all have read it. A read behind the last barrier of a unit would see the next unit's flag, and the
    waves of a work-group could part at the barriers under it."""
    text = open(os.path.join(PKG, "csrc", "mdx_paged_attn.hip")).read()
    body = text[text.index("void paged_attn_kernel"):text.index("void paged_join_kernel")]
    ring_free = body.index("// the ring is free")
    body = re.sub(r"//[^\n]*", lambda m: " " * len(m.group()), body)
    next_barrier = body.index("__syncthreads", ring_free)
    reads = []
    for m in re.finditer(r"\bodd\b(\[[^\]]*\])?", body):
        line = body[body.rindex("\n", 0, m.start()) + 1:m.start()]
        declared = "__shared__" in line
        written = re.match(r"\s*=[^=]", body[m.end():]) or re.search(r"atomic(Min|Max)\(&?$", line)
        if not declared and not written:
            reads.append(m.start())
    assert reads and all(ring_free < r < next_barrier for r in reads), [body[r - 40:r + 20] for r in reads]
