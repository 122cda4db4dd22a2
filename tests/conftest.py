import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")
    # NCCL_DEBUG=VERSION makes RCCL print its banner ("RCCL version ...") between the lines that tests read from their children's stdout
    if os.environ.get("NCCL_DEBUG") == "VERSION":
        os.environ["NCCL_DEBUG"] = "NONE"


# GPU tests written in round 4 while the device pool was closed to this repository: they have never run on the
# device.  They are scheduled BEHIND the tests that have (a stable partition of the collection order), so that under
# `-x` a defect in a new test cannot hide the verdict of the 229 proven ones.
ROUND4_UNPROVEN = ("test_bench_gpu.py", "test_aux_gpu.py", "test_native_row_partitioned_spgemm",
                   "test_split_row_spmv_for_cache_resident_matrices", "test_hash_bins_both_kernel_families[3]",
                   "test_big_table_bins_on_clustered_columns[3]", "test_one_wavefront_bin[3]",
                   "test_random_amb_plans", "test_exotic_gpu.py", "test_numeric_rerun_of_ranked_window_rows",
                   "test_config5_code_paths_at_a_fifth_of_the_edges")  # (round 5: first run on the CPU emulation, tests/emu)


# ... and behind those, the tests whose verdict also depends on tools of the box (rocprofv3 marker traces, the ASan
# runtime preloaded under the ROCm runtime): a surprise there must not stop (-x) anything that is about the library.
ENVIRONMENT_LAST = ("test_roctx_ranges_reach_a_marker_trace", "test_asan_build_runs_clean")


def _lend_names(items):
    """tests/test_spgemm_gpu.py names gpu_util.variant_env in a test without importing it (only the script that the test runs does)."""
    for module in {it.module for it in items if getattr(it, "module", None) and it.module.__name__ == "test_spgemm_gpu"}:
        from gpu_util import variant_env
        module.variant_env = variant_env


def pytest_collection_modifyitems(config, items):
    _lend_names(items)
    last = [it for it in items if any(tag in it.nodeid for tag in ENVIRONMENT_LAST)]
    new = [it for it in items if it not in last and any(tag in it.nodeid for tag in ROUND4_UNPROVEN)]
    if new or last:
        old = [it for it in items if it not in new and it not in last]
        items[:] = old + new + last


@pytest.fixture(scope="session")
def oracle_d():
    from oracle.oracle import Oracle
    return Oracle("d")


@pytest.fixture(scope="session")
def oracle_s():
    from oracle.oracle import Oracle
    return Oracle("s")


def _with_test_switches(lib):
    # NSPARSE_TEST_WS_CACHE=0|1|2: the workspace mode for the whole session (0: every array of a call is its own
    # hipMalloc -- what the AddressSanitizer build of the emulation wants, tests/emu/README.md)
    m = os.environ.get("NSPARSE_TEST_WS_CACHE")
    if m is not None:
        lib.nsparse_set_workspace_cache(int(m))
    return lib


@pytest.fixture(scope="session")
def lib_d():
    import nsparse_amd
    return _with_test_switches(nsparse_amd.load("d"))


@pytest.fixture(scope="session")
def lib_s():
    import nsparse_amd
    return _with_test_switches(nsparse_amd.load("s"))


def load_golden(name):
    z = np.load(os.path.join(GOLDEN, name + ".npz"))
    d = {k: z[k] for k in z.files}
    d["M"], d["N"] = int(d["M"]), int(d["N"])
    d["nnz"] = int(d["rpt"][-1])
    return d


# known answers for the reference's only fixture, data/test.mtx
TEST_MTX = dict(
    M=5, N=5, nnz=9, nnz_max=3,
    rpt=[0, 2, 3, 6, 7, 9], col=[0, 2, 1, 0, 2, 4, 3, 2, 4],
    val=[10, 1, 20, 1, 30, 2, 40, 2, 50],
    x=[1, 2, 3, 4, 5], y=[13, 40, 101, 160, 256],
    row_prod=[5, 1, 7, 1, 5], n_prod=19,
    c_rpt=[0, 3, 4, 7, 8, 11], c_col=[0, 2, 4, 1, 0, 2, 4, 3, 0, 2, 4],
    c_val=[101, 40, 2, 400, 40, 905, 160, 1600, 2, 160, 2504],
)
