"""Copies in flight end before their CTA does, also where a wait ran out: a thread that lands them only if the CTA's abort flag is up reads the flag behind a
barrier of the whole CTA that follows every wait, else a wait that runs out later would leave them in flight.  Read from the source: such a wait must not be
made to run out on a GPU."""
import os
import re

import pytest

from test_cluster_stores_host import CSRC, functions

FILES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and "mb_land_ring(" in open(os.path.join(CSRC, f)).read() and f != "mbarrier.cuh")
WAIT = re.compile(r"\bmb_wait\w*\(")
LAND = re.compile(r"\bmb_land_ring\(")


def top_level(body):
    """The body with everything inside braces and the statements behind conditions and loops blanked, at the same length."""
    out, depth = [], 0
    for c in body:
        depth += c == "{"
        out.append(c if depth == 0 else " ")
        depth -= c == "}"
    return re.sub(r"\b(?:if|for|while|else)\b[^;]*;", lambda m: " " * len(m.group(0)), "".join(out))


def early_looks(source):
    """Kernels that decide by the abort flag whether to land their copies without a barrier between the last wait and that look."""
    found = []
    for name, body, kernel in functions(source):
        lands = [m.start() for m in LAND.finditer(body)] if kernel else []
        flags = [m.start() for m in re.finditer(r"if \([^;{]*abort_flag\)", body)]
        # a landing is conditional if the flag's condition opens its block, or its statement
        conditional = [f for f in flags if any(f < at and (";" not in body[f:at] or body[f:at].count("{") > body[f:at].count("}")) for at in lands)]
        for look in conditional:
            last = max((m.start() for m in WAIT.finditer(body) if m.start() < look), default=0)
            if not re.search(r"__syncthreads\(\);", top_level(body)[last:look]):
                found.append(name)
    return found


def test_files_are_found():
    assert {"mx4_gemv.cu", "image_gemm.cu", "gemm_wide.cu"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_copies_land_behind_a_barrier_or_always(name):
    with open(os.path.join(CSRC, name)) as f:
        assert early_looks(f.read()) == []


def test_the_reader_finds_a_look_in_front_of_the_barrier():
    kernel = "__global__ void k(const Args a) {\n    for (int i = 0; i < n; ++i) {\n        if (!mb_wait(&full[i], 0, a.err, &sh.abort_flag)) continue;\n        %s\n    }\n    %s\n    if (%ssh.abort_flag) %s\n}\n"
    land = "mb_land_ring(sh.full, n, 4);"
    assert early_looks(kernel % ("", "__syncthreads();", "", land)) == []
    assert early_looks(kernel % ("", "__syncthreads();", "tid == 0 && ", "{ if (warp == 0) " + land + " }")) == []
    assert early_looks(kernel % ("", "", "tid == 0 && ", land)) == ["k"]
    assert early_looks(kernel % ("__syncthreads();", "", "", "{ if (warp == 0) " + land + " }")) == ["k"]
    assert early_looks(kernel % ("", "if (a.split > 1) __syncthreads();", "", land)) == ["k"]
    assert early_looks(kernel % ("", land, "", "x = 1;")) == []
