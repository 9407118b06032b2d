"""A rule that the kernels' sources keep and that no result shows."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'gc_moe_b200', 'csrc')


def test_no_non_coherent_loads():
    """Every kernel may start while the one before it still writes (programmatic dependent launch), so no memory is
    read-only for a kernel's lifetime, which the non-coherent path asks for."""
    sources = glob.glob(os.path.join(CSRC, '*.cu*'))
    assert len(sources) > 5
    for path in sources:
        code = re.sub(r'//[^\n]*', '', open(path).read())
        assert '__ldg' not in code and not re.search(r'ld\.global(\.\w+)*\.nc', code), path
