"""Kernels of caches and rotations keep everything in registers: no scratch memory.  Read from the built library's metadata."""
from test_kernel_registers import _scratch_bytes


def test_caches_and_rotations_spill_nothing(tmp_path):
    found = _scratch_bytes(tmp_path)
    for family, least in (("5cache12_GLOBAL__N_116attention_kernel", 40), ("join_shares_kernel", 9), ("12write_kernel", 18), ("11read_kernel", 18), ("13rotate_kernel", 18),
                          ("22rotate_backward_kernel", 18), ("14weights_kernel", 9)):
        kernels = {k: v for k, v in found.items() if family in k}
        assert len(kernels) >= least, (family, len(kernels))
        assert {k: v for k, v in kernels.items() if v} == {}, family
