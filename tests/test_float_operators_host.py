"""Host-side checks of the float operators' sources and helpers that need no device."""
import os
import re

from spatialdb_b200 import build


def source(name):
    text = open(os.path.join(build.CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_dependents_start_after_the_tensor_memory_is_taken():
    """A kernel that may run beside this one must find its tensor memory taken: every CTA of the product allocates,
    meets at a barrier, and only then lets dependents start."""
    body = source("k_linear_tc.cu")
    body = body[body.index("k_linear_tc(const __grid_constant__"):]
    alloc = [m.start() for m in re.finditer(r"tcgen05\.alloc\.", body)]
    release = [m.start() for m in re.finditer(r"grid_release\(\)", body)]
    assert len(alloc) == 2 and len(release) == 1
    barrier = body.index("__syncthreads()", max(alloc))
    assert max(alloc) < barrier < release[0] < body.index("grid_wait()")
