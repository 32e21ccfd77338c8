"""First calls from several threads at once, without a GPU: what the host part of a call looks up once (csrc/tcgen05.cuh) is there for every thread that asks."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.metal_b200", "csrc")

STANDIN = """
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
enum cudaError_t { cudaSuccess };
enum cudaDriverEntryPointQueryResult { cudaDriverEntryPointSuccess };
enum { cudaEnableDefault };
typedef int (*encode_fn_t)();
static int asked = 0;
static int answer() { return 0; }
static cudaError_t cudaGetDriverEntryPoint(const char *, void **p, int, cudaDriverEntryPointQueryResult *q)
{
    ++asked;
    std::this_thread::sleep_for(std::chrono::milliseconds(100));
    *p = reinterpret_cast<void *>(answer);
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
%s
int main()
{
    std::vector<std::thread> all;
    encode_fn_t got[8];
    for (int i = 0; i < 8; ++i) all.emplace_back([&, i] { got[i] = encode_fn(); });
    for (auto &t : all) t.join();
    int there = 0;
    for (auto f : got) there += f == answer;
    printf("%%d %%d", there, asked);
}
"""


def test_every_thread_gets_the_entry_point(tmp_path):
    with open(os.path.join(CSRC, "tcgen05.cuh")) as f:
        s = f.read()
    at = s.index("inline encode_fn_t encode_fn()")
    source, exe = tmp_path / "first.cpp", str(tmp_path / "first")
    source.write_text(STANDIN % s[at:s.index("\n}\n", at) + 3])
    subprocess.run(["g++", "-O1", "-std=c++17", "-pthread", str(source), "-o", exe], check=True)
    assert subprocess.run([exe], check=True, stdout=subprocess.PIPE, text=True, timeout=60).stdout == "8 1"
