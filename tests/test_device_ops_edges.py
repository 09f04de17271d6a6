"""Operators over device buffers at the edges of what their calls allow, without a device."""
import re

from test_dependent_launches import kernels


def test_kernels_have_their_tensor_memory_before_the_next_may_start():
    """The next kernel may take tensor memory and wait for this one's end: if this one still waited for that memory, neither would end."""
    seen = 0
    for file, name, _, body in kernels():
        takes = re.search(r"tmem_alloc\(|tcgen05\.alloc", body)
        if takes and "pdl_trigger()" in body:
            seen += 1
            assert body.rindex("tmem_alloc(" if "tmem_alloc(" in body else "tcgen05.alloc") < body.index("pdl_trigger()"), (file, name)
    assert seen >= 4
