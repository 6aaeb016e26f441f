"""CPU: a kernel that allocates tensor memory lets the next kernel of its stream in only from the warp that has been given it, or behind a barrier with
that warp.  (The next kernel may hold columns until this one is complete: let in earlier, it could take those that this one still waits for.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "f2cgt_b200", "csrc")
ALLOCATES = re.compile(r"\balloc_tmem(?:_pair)?\(|tcgen05\.alloc\.")
RELEASES = "release_dependents();"


def text(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def kernels():
    """(name, body) of the kernels that allocate, with the function that the k-means kernels share in its place"""
    shared = text("kmeans_tc.cuh")
    run = shared[shared.index("bool NO_WAITS, typename P>"):]
    for file in sorted(f for f in os.listdir(CSRC) if f.endswith(".cu")):
        for part in text(file).split("__global__")[1:]:
            part = part[:part.index("\n}\n")].replace("run<C, NB, NO_WAITS>(p);", run)
            if ALLOCATES.search(part):
                yield re.search(r"(\w+_kernel)\(", part).group(1), part


FOUND = dict(kernels())


def block_of(body, at):
    """where the innermost braces around `at` open"""
    depth = 0
    for i in range(at, -1, -1):
        depth += {"}": 1, "{": -1}.get(body[i], 0)
        if depth < 0:
            return i
    return 0


def test_the_kernels_are_known():
    assert set(FOUND) == {"sage_forward_kernel", "kmeans_tc_kernel", "kmeans_fit_kernel", "mm_kernel", "linear_kernel", "product_kernel", "small_kernel"}


@pytest.mark.parametrize("name", sorted(FOUND))
def test_release_follows_allocation(name):
    body = FOUND[name]
    last = [m.end() for m in ALLOCATES.finditer(body)][-1]
    for m in re.finditer(re.escape(RELEASES), body):
        assert m.start() > last
        if "__syncthreads();" in body[last:m.start()]:
            continue
        lead = body[:m.start()].rstrip()
        own_warp = re.search(r"if \((wid == \d)\)$", lead)
        if own_warp:
            assert re.search(r"if \(" + own_warp.group(1) + r"\) (?:\{\s*)?alloc_tmem", body)
        else:
            opens = block_of(body, last)  # the block of that warp alone
            assert block_of(body, m.start()) == opens and re.search(r"if \((?:wid|warp) == \w+\) $", body[:opens])
