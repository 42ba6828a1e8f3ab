"""The kernels' loads of words that are no whole vector, on the CPU: against the
end of readable memory."""
import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "pjrtx_amd" / "csrc"

MAIN = r"""
#include "kernels/vec.h"
#include <cstdio>
#include <cstring>
#include <sys/mman.h>
#include <unistd.h>

// The last N words before a page that must not be read, at 2 bytes' alignment
// and at 4.
template <int N>
static int check(char* end) {
  int bad = 0;
  for (int back = 0; back <= 2; back += 2) {
    uint32_t want[N], got[N];
    for (int i = 0; i < N; ++i) want[i] = 0x01020304u * (i + 1) + back;
    std::memcpy(end - back - 4 * N, want, 4 * N);
    pjrtx::load_words<N>(end - back - 4 * N, got);
    bad += std::memcmp(got, want, 4 * N) != 0;
  }
  return bad;
}

int main() {
  const size_t page = sysconf(_SC_PAGESIZE);
  char* p = static_cast<char*>(mmap(nullptr, 2 * page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
  if (p == MAP_FAILED || mprotect(p + page, page, PROT_NONE)) return 2;
  return check<1>(p + page) + check<2>(p + page) + check<3>(p + page) + check<4>(p + page);
}
"""


@pytest.mark.parametrize("level", ["-O0", "-O3"])
def test_loads_of_words_read_no_byte_past_them(tmp_path, level):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not pathlib.Path(hipcc).exists():
        pytest.skip("no hipcc")
    (tmp_path / "main.hip").write_text(MAIN)
    cmd = [hipcc, "-std=c++17", level, "-x", "hip", "--offload-host-only", "-I", str(CSRC), str(tmp_path / "main.hip"),
           "-o", str(tmp_path / "main")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert subprocess.run([str(tmp_path / "main")]).returncode == 0
