"""The table of the LDS that kernels have reserved: each kernel's attribute is set
once per size that is larger than before, however many kernels there are and from
several threads (no GPU: the HIP call is a stub that counts)."""
import os
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "teco-ops_amd", "csrc")

PROGRAM = r"""
#include "handle.cpp"

#include <cstdlib>
#include <thread>
#include <vector>

static std::atomic<int> sets{0};
static int refuse = 0;
extern "C" hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int) {
    ++sets;
    return refuse ? hipErrorInvalidValue : hipSuccess;
}
extern "C" hipError_t hipGetLastError() { return hipSuccess; }

static void expect(int n, const char *what) {
    if (sets == n) return;
    std::printf("%s: %d sets for %d\n", what, sets.load(), n);
    std::exit(1);
}

int main() {
    const int N = 700;
    static char kernels[N * 16 + 1];
    const auto at = [&](int i) { return static_cast<const void *>(kernels + i * 16); };
    const auto all = [&](size_t bytes) {
        for (int i = 0; i < N; ++i)
            if (!tecoops::reserve_lds(at(i), bytes)) std::exit(2);
    };
    all(64 * 1024);
    expect(0, "the default");
    for (int turn = 0; turn < 3; ++turn) all(100 * 1024);
    expect(N, "once each");
    all(80 * 1024);
    expect(N, "less than before");
    all(160 * 1024);
    all(100 * 1024);
    expect(2 * N, "more than before");
    if (tecoops::reserve_lds(at(0), 160 * 1024 + 1)) return 3;
    refuse = 1;
    static char other;
    if (tecoops::reserve_lds(&other, 100 * 1024)) return 4;
    refuse = 0;
    if (!tecoops::reserve_lds(&other, 100 * 1024) || !tecoops::reserve_lds(&other, 100 * 1024)) return 5;
    expect(2 * N + 2, "refused, then set");
    // eight threads over new kernels: one set each
    static char more[N * 16];
    std::vector<std::thread> threads;
    for (int t = 0; t < 8; ++t)
        threads.emplace_back([&, t] {
            for (int i = 0; i < 2 * N; ++i)
                if (!tecoops::reserve_lds(more + (i + 97 * t) % N * 16, 70 * 1024)) std::exit(6);
        });
    for (auto &t : threads) t.join();
    expect(3 * N + 2, "threads");
    return 0;
}
"""


def test_each_kernel_is_set_once(tmp_path):
    src, exe = tmp_path / "lds.cpp", tmp_path / "lds"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__=1", "-pthread", "-I", CSRC, "-I",
                    os.path.join(REPO, "include"), "-I", "/opt/rocm/include", str(src), "-o", str(exe), "-L",
                    "/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)
