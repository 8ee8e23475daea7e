"""A failed runtime call is reported once: by the entry point that made it, not again by the next launch."""
import os
import subprocess

from conftest import ROOT

# the library's own checks around a runtime that is written here: it keeps an error until it is asked for
PROGRAM = r"""
#include "common.h"
static hipError_t kept = hipSuccess;
extern "C" hipError_t hipGetLastError() { hipError_t e = kept; kept = hipSuccess; return e; }
extern "C" const char* hipGetErrorString(hipError_t) { return "refused"; }
namespace mpnn { char* error_buffer() { static char text[512]; return text; } }
static hipError_t refused() { return kept = hipErrorInvalidValue; }
static int32_t attribute() { MPNN_HIP_CHECK(refused()); return MPNN_OK; }
static int32_t launch() { MPNN_LAUNCH_CHECK("k"); return MPNN_OK; }
int main() {
  if (launch() != MPNN_OK) return 1;
  if (attribute() != MPNN_E_HIP || !strstr(mpnn::error_buffer(), "refused() failed: refused")) return 2;
  if (launch() != MPNN_OK) return 3;
  kept = hipErrorInvalidValue;
  if (launch() != MPNN_E_HIP || !strstr(mpnn::error_buffer(), "launch of k failed")) return 4;
  return launch() == MPNN_OK ? 0 : 5;
}
"""


def test_an_error_is_reported_once(tmp_path):
    source, program = tmp_path / "errors.cpp", tmp_path / "errors"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I", os.path.join(ROOT, "mpnn_amd", "csrc"),
                    str(source), "-o", str(program)], check=True, capture_output=True)
    assert subprocess.run([str(program)]).returncode == 0
