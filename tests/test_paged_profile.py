"""The profiling harness on the rope and paged-cache kernels (no GPU needed)."""

import os
import sys

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(_REPO, "flash-attention-cuda_amd", "profile"))

import profile_workload as pw  # noqa: E402
import rocprof_extract as rx  # noqa: E402


def test_kernels_of_both_types_stay_apart():
    name = "_ZN2fa12_GLOBAL__N_119attend_paged_kernelI{}Li128EEEvNS_17AttendPagedParamsE"
    assert rx.short_kernel_name(name.format("DF16_")) == "attend_paged_kernel<_Float16, 128>"
    assert rx.short_kernel_name(name.format("DF16b")) == "attend_paged_kernel<__bf16, 128>"
    assert rx.short_kernel_name(
        "_ZN2fa12_GLOBAL__N_111rope_kernelIDF16bLb1EEEvNS0_10RopeParamsE") == \
        "rope_kernel<__bf16, true>"


def test_every_workload_has_a_runner_and_states_its_work():
    assert set(pw.WORKLOADS) == set(pw.RUNNERS)
    lens = pw._decode_inputs(32, 1, 4096)[3]
    assert int(lens.sum()) == 73374  # of decode_c5, decode_gqa_c5 and attend_batch
    assert sum(1024 * i - 1 for i in range(1, 9)) == 36856  # of attend_long
    assert pw.WORKLOADS["attend_chunks"][3] == 4.0 * 4 * 32 * 128 * sum(range(6145, 8193))
