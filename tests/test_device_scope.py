"""A library call made while another device is current (csrc/device_scope.h): the scope switches once,
restores the caller's device once, and does nothing where the device is already right.  Built for the
host with stand-ins for the two runtime calls (no GPU needed)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "device_scope.h"
static int current = 1, gets = 0, sets = 0;
extern "C" hipError_t hipGetDevice(int* d) {
    if (++gets > 16) { std::puts("does not end"); std::exit(3); }
    *d = current;
    return hipSuccess;
}
extern "C" hipError_t hipSetDevice(int d) {
    if (d > 7) return hipErrorInvalidDevice;
    if (++sets > 16) { std::puts("does not end"); std::exit(3); }
    current = d;
    return hipSuccess;
}
#define EXPECT(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
    {
        lily::DeviceScope a(0);
        EXPECT(a.err == hipSuccess && current == 0 && sets == 1);
        {
            lily::DeviceScope b(0);   // a call made by a call
            EXPECT(b.err == hipSuccess && current == 0 && sets == 1);
        }
        EXPECT(current == 0 && sets == 1);
    }
    EXPECT(current == 1 && sets == 2);
    { lily::DeviceScope c(1); }
    EXPECT(current == 1 && sets == 2);
    { lily::DeviceScope d(9); EXPECT(d.err == hipErrorInvalidDevice); }
    EXPECT(current == 1 && sets == 2);
    std::puts("ok");
    return 0;
}
"""


def test_a_call_leaves_the_thread_on_its_device(tmp_path):
    src, exe = tmp_path / "scope.cpp", tmp_path / "scope"
    src.write_text(PROGRAM)
    csrc = os.path.join(ROOT, "lily-qwen3.8-flash-next_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", csrc, "-I", "/opt/rocm/include",
                    str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout
