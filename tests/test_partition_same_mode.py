"""Setting the partition mode that a device is in already: nothing to do, and
no privilege to ask for. Against a stand-in for the management library that
has no setters."""
import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

LIBRARY = r"""
#include <cstdint>
#include <cstdio>
#include <cstring>
static int one;
extern "C" {
int amdsmi_init(uint64_t) { return 0; }
int amdsmi_shut_down() { return 0; }
int amdsmi_get_socket_handles(uint32_t* n, void** s) {
  *n = 1;
  if (s) s[0] = &one;
  return 0;
}
int amdsmi_get_processor_handles(void*, uint32_t* n, void** p) {
  *n = 1;
  if (p) p[0] = &one;
  return 0;
}
int amdsmi_get_gpu_device_uuid(void*, unsigned* n, char* u) {
  snprintf(u, *n, "GPU-stand-in");
  return 0;
}
int amdsmi_get_gpu_memory_total(void*, int, uint64_t* b) { *b = 1; return 0; }
int amdsmi_get_gpu_memory_usage(void*, int, uint64_t* b) { *b = 0; return 0; }
int amdsmi_get_gpu_activity(void*, void*) { return 1; }
int amdsmi_get_gpu_process_list(void*, uint32_t* n, void*) { *n = 0; return 0; }
int amdsmi_get_gpu_bdf_id(void*, uint64_t* b) { *b = 1; return 0; }
int amdsmi_get_gpu_compute_partition(void*, char* m, uint32_t n) {
  snprintf(m, n, "SPX");
  return 0;
}
int amdsmi_get_gpu_memory_partition(void*, char* m, uint32_t n) {
  snprintf(m, n, "NPS1");
  return 0;
}
}
"""

PROGRAM = """
from tensor_fusion_amd.hypervisor.device import Accelerator
a = Accelerator()
assert a.devices()[0].uuid == "GPU-stand-in", a.devices()
assert (a.compute_partition(0), a.memory_partition(0)) == ("SPX", "NPS1")
assert a.set_compute_partition(0, "SPX") and a.set_compute_partition(0, "spx")
assert a.set_memory_partition(0, "NPS1")
assert not a.set_compute_partition(0, "CPX")
assert not a.set_memory_partition(0, "NPS4")
for change in (lambda: a.set_compute_partition(0, "BOGUS"),
               lambda: a.set_memory_partition(0, "NPS3"),
               lambda: a.set_compute_partition(1, "SPX")):
    try:
        change()
    except RuntimeError:
        continue
    raise AssertionError("not refused")
"""


@pytest.mark.usefixtures("native_built")
def test_the_mode_it_is_in(tmp_path):
    src = tmp_path / "smi.cpp"
    src.write_text(LIBRARY)
    subprocess.run(["g++", "-shared", "-fPIC", str(src), "-o",
                    str(tmp_path / "libamd_smi.so")], check=True)
    env = dict(os.environ, LD_LIBRARY_PATH=str(tmp_path))
    env.pop("TF_ACCEL_MOCK", None)
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=REPO, env=env,
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
