"""The same for the kernels of a text stage: what their loads into shared memory rest on, and registers, of which their occupancy is. CPU only."""

import re

import pytest

from test_device_code import _assembly, _functions, _registers, _written_in_front


def _loads_to_lds(code):
    return [i for i, text in enumerate(code) if text.startswith("buffer_load") and text.endswith("lds") or text.startswith("global_load_lds")]


def test_ruled_loads_wait_for_their_scalar_registers():
    """A memory instruction may read a scalar register 5 wait states after a vector instruction has written it and no sooner."""
    kernels = _functions("attn_ruled.hip", labels=True)
    mains = [name for name in kernels if "attn_ruled_kernel" in name]
    assert len(mains) == 48  # 2 types, 2 head sizes, with and without a cap, 3 biases, 2 ways to share a tile
    for name in mains:
        code = kernels[name]
        loads = _loads_to_lds(code)
        assert len(loads) >= 9, name
        for at in loads:
            scalars = {r for o in re.split(r"[,\s]+", code[at]) for r in _registers(o) if r[0] == "s"}
            assert len(scalars) >= 4, code[at]
            assert code[at - 2].startswith("s_mov_b32 m0") and code[at - 1] == "s_nop 3", (name, code[at - 2:at + 1])
            assert _written_in_front(code, at, scalars, 5) is None, (name, code[at - 8:at + 1])


def test_paged_loads_follow_their_destination_and_the_reads_of_their_stage():
    """m0 is written one wait state ahead of a load that takes its destination from there, and no load of the loop goes out while reads from
    shared memory are on their way: the stage that it fills is the one that was read last."""
    kernels = _functions("attn_paged.hip")
    mains = [name for name in kernels if "attn_paged_kernel" in name]
    assert len(mains) == 24
    for name in mains:
        code = kernels[name]
        loads = _loads_to_lds(code)
        assert len(loads) >= 8, name
        for at in loads:
            assert code[at - 2].startswith("s_mov_b32 m0") and code[at - 1] == "s_nop 0", (name, code[at - 2:at + 1])
            behind = [i for i in range(at) if code[i].startswith("ds_read") and "tr_b16" in code[i]]  # (the values' reads, a tile's last)
            if behind:
                assert any(text.startswith("s_waitcnt") and "lgkmcnt(0)" in text for text in code[behind[-1]:at]), (name, code[at])


@pytest.mark.parametrize("source,kernel,most,scratch", [
    ("attn_ruled.hip", "attn_ruled_kernelI.*Li64E", 168, 8), ("attn_ruled.hip", "attn_ruled_kernelI.*Li128E", 256, 0),  # 3 and 2 wavefronts to a SIMD
    ("attn_paged.hip", "attn_paged_kernelI.*Li64E", 128, 0), ("attn_paged.hip", "attn_paged_kernelI.*Li128E", 256, 0),  # 4 and 2
    ("rope_append.hip", "rope_append_kernel", 64, 0)])                                                                  # 8
def test_registers_leave_the_occupancy_that_the_kernels_count_on(source, kernel, most, scratch):
    name, found = None, {}
    for line in _assembly(source):
        if line.startswith(".amdhsa_kernel "):
            name = line.split()[1]
        elif line.startswith((".amdhsa_next_free_vgpr ", ".amdhsa_private_segment_fixed_size ")):
            found.setdefault(name, {})[line.split()[0]] = int(line.split()[1])
    found = {k: v for k, v in found.items() if re.search(kernel, k)}
    assert len(found) >= 6
    for k, v in found.items():
        assert v[".amdhsa_next_free_vgpr"] <= most and v[".amdhsa_private_segment_fixed_size"] <= scratch, (k, v)
