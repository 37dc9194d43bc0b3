"""No kernel of the cache and of attention over it or in windows spills registers, whatever the head size."""
import tensorrt_amd
from test_kernel_resources_host import code_objects, kernels


def test_no_attention_kernel_spills():
    found = {}
    with open(tensorrt_amd.library_path(), "rb") as f:
        for elf in code_objects(f.read()):
            found.update((k[".name"], k) for k in kernels(elf))
    ours = [k for n, k in found.items() if any(x in n for x in ("cached_", "window_attention", "kv_cache"))]
    assert len(ours) > 60
    spilling = {k[".name"]: k[".vgpr_spill_count"] for k in ours if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not spilling
