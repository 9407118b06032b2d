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


def test_tensor_memory_is_allocated_before_dependents_may_start():
    """A dependent that holds tensor memory of the SM waits for the end of the kernel that let it start; an allocation
    behind that point could wait for the dependent, without end."""
    found = 0
    for path in glob.glob(os.path.join(CSRC, '*.cuh')):
        code = re.sub(r'//[^\n]*', '', open(path).read())
        if path.endswith('ptx.cuh') or 'ptx::tmem_alloc' not in code:
            continue
        body = code[code.rindex('__global__', 0, code.rindex('ptx::tmem_alloc')):]
        assert body.index('ptx::tmem_alloc') < body.index('ptx::launch_dependents'), path
        found += 1
    assert found == 2
