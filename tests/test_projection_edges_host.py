"""Host-side checks at the edges of the 8-bit projections and the orthogonalised
steps (no GPU needed)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fg-cpab_b200", "csrc")


def code_of(name):
    """A source file without its comments."""
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", sorted(n for n in os.listdir(CSRC) if n.endswith((".cu", ".cuh"))))
def test_kernels_that_begin_early_read_with_ordinary_loads(name):
    """A kernel that waits for the one before (griddepcontrol.wait) runs while that
    one writes: read-only loads may return what was there before."""
    code = code_of(name)
    if not re.search(r"griddepcontrol\.wait|\bdep_wait\b", code):
        pytest.skip("no kernel of this file begins early")
    assert not re.findall(r"__ldg|ld\.global(?:\.\w+)*\.nc|__restrict__", code)
