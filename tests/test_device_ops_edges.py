"""Operators over device buffers at the edges of what their calls allow, without a device."""
import re

from test_dependent_launches import kernels

# more than 860 threads and 180 KB of shared memory: no CTA that wants tensor memory fits beside one of these
ALONE_ON_AN_SM = {"qstream_tc_kernel"}


def test_kernels_have_their_tensor_memory_before_the_next_may_start():
    """The next kernel may take tensor memory and wait for this one's end: if this one still waited for that memory, neither would end."""
    seen = set()
    for file, name, _, body in kernels():
        takes = [m.start() for m in re.finditer(r"tmem_alloc\(|tcgen05\.alloc", body)]
        if takes and "pdl_trigger()" in body and name not in ALONE_ON_AN_SM:
            seen.add(name)
            assert takes[-1] < body.index("pdl_trigger()"), (file, name)
    assert {"shared_keys_kernel", "attn_umma_kernel", "hgemm_tc_kernel", "latent_umma_kernel"} <= seen
