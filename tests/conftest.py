import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    config.addinivalue_line("markers", "slow: long-running test")


# GPU tests of what KFD shows of each process: its VRAM and queues (host truth, amd-smi's process list) and its resident
# waves, from which the share-board sampler charges governed tenants.  Where a machine hides that directory they have
# nothing to measure: the sampler does not start, and the governor charges wall time instead of shares.
KFD_PROC = Path("/sys/class/kfd/kfd/proc")
NEEDS_KFD_PROC = {
    "test_a8_tenants_gpu.py": {"test_eight_temporal_tenants_run_like_native",
                               "test_eight_pooled_slices_with_the_monitor_switch"},
    "test_e2e_gpu.py": {"test_pod_on_mi355x_end_to_end", "test_time_sharing_mode_on_the_real_node",
                        "test_shimless_container_on_time_shared_gpu_is_evicted"},
    "test_partition_gpu.py": {"test_manager_never_reconfigures_a_gpu_in_use"},
    "test_shim_gpu.py": {"test_runtime_vram_charged_as_context", "test_temporal_slices_charged_the_share_they_receive",
                         "test_unequal_temporal_limits_get_their_shares",
                         "test_four_symmetric_temporal_tenants_run_like_native"},
    "test_shim_interpose_gpu.py": {"test_triton_kernel_loop_held_to_its_share",
                                   "test_module_bytes_reported_and_kfd_split_exact",
                                   "test_granted_queue_cap_holds_against_the_tenant",
                                   "test_tenant_without_the_shim_reported_within_one_pass",
                                   "test_tenant_rewriting_its_region_cannot_unblock_itself"},
}


def pytest_collection_modifyitems(items):
    if KFD_PROC.is_dir():
        return
    skip = pytest.mark.skip(reason=f"not run: KFD shows no processes on this machine ({KFD_PROC} is missing)")
    for item in items:
        if getattr(item, "originalname", None) in NEEDS_KFD_PROC.get(item.path.name, ()):
            item.add_marker(skip)


@pytest.fixture(scope="session")
def native_build():
    """Build the shim + mock HIP runtime once per session (CPU-safe)."""
    from k8s_vgpu_scheduler_amd.utils import build
    build.build_shim()
    mock_lib, driver = build.build_mock()
    return {"shim": build.SHIM_SO, "mock_lib": mock_lib, "driver": driver, "roctx": build.MOCK_ROCTX,
            "boardd": build.build_boardd(), "mock_smi": build.MOCK_SMI}
