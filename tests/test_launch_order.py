"""The paged kernels start while the kernel before them still runs (programmatic dependent launch). What keeps that sound is
the order of a few calls in their sources, which is checked here, by reading them: no test on a GPU shows it."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vsa_lm_b200", "csrc")
FILES = ("paged.cu", "paged_attend.cu", "paged_prompt.cu")


def _kernels():
    """(file, name, body without comments) of every kernel of the files."""
    out = []
    for f in FILES:
        src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, f)).read())
        for m in re.finditer(r"__global__ void[^{;]*?(\w+)\(const __grid_constant__", src):
            body = src[m.end():src.index("\n}\n", m.end())]
            out.append((f, m.group(1), body))
    return out


KERNELS = _kernels()


def test_all_kernels_are_found():
    assert len(KERNELS) == sum(open(os.path.join(CSRC, f)).read().count("__global__") for f in FILES) >= 10


@pytest.mark.parametrize("f,name,body", KERNELS, ids=[k[1] for k in KERNELS])
def test_a_kernel_waits_before_it_reads_what_earlier_ones_wrote(f, name, body):
    """One wait, by all threads, before lengths, table, pages, queries, records or the workspace are touched."""
    waits = [m.start() for m in re.finditer(r"grid_dep_wait\(\);", body)]
    assert len(waits) == 1 and re.search(r"\n  grid_dep_wait\(\);\n", body)
    reads = re.search(r"\blen\.rows\(|\bpage_of\(|\bcopy_queries<|\btma_load|\bcp_async16\(|\ba\.(lens|weight|order|table|status)\b"
                      r"|\bp\.(part|part_ml|lse|span|count|moves)\[|\bparts_of\(|\btoken_at\(|\bload_norms<|\b__ldg\(|\bmove_rows<", body)
    assert reads and waits[0] < reads.start(), body[reads.start():reads.start() + 40]


@pytest.mark.parametrize("f,name,body", [k for k in KERNELS if "tmem_alloc(" in k[2]], ids=[k[1] for k in KERNELS if "tmem_alloc(" in k[2]])
def test_a_kernel_has_its_tensor_memory_before_the_next_one_starts(f, name, body):
    """Else a block of the next kernel could take the columns on the same SM and wait, with them, for this grid's end. And it
    takes none before its own wait, which the kernels before it could need."""
    assert body.count("grid_dep_launch();") == body.count("tmem_alloc(") == 1
    assert body.index("grid_dep_wait();") < body.index("tmem_alloc(") < body.index("grid_dep_launch();")
