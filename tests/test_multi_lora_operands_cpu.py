"""Where the adapters' row sums read their operands, on the host: every 16 bytes that a wave
loads lie inside the buffer that the size queries ask for, whatever the rank."""
import ctypes
import os
import subprocess
import sys

import pytest

from rocm_qlora import _native as nat

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocm-qlora_amd", "csrc")
INCLUDE = os.path.join(os.path.dirname(os.path.dirname(CSRC)), "include")

# the loads of rowsum's waves over the last 32 slots of `slots`: the largest byte past the start,
# and how many of a rank's operands a wave loads from another rank's place (of ranks that count)
SOURCE = r"""
#include <cstdio>
#include "rq_multi_lora.h"
using namespace rq;
template <int XT>
void reach(int r, long slots) {
  constexpr int es = XT == RQ_DTYPE_F32 ? 4 : 2;
  const int rp = int(rank_pad(r)), jb = rowsum_blocks(rp);
  long most = 0, wrong = 0;
  for (int j0 = 0; j0 < rp; j0 += 16 * jb)
    for (int j = 0; j < jb; ++j)
      for (int lane = 0; lane < 64; ++lane) {
        const int i = lane & 15, g = lane >> 4, from = rowsum_rank(j0, j, rp);
        const int64_t at = opt_at<XT>(8 * g, i, rp) + opt_at<XT>(slots - 32, from, rp);
        for (int p = 0; p < 2; ++p) {
          const int64_t last = es * (at + (XT == RQ_DTYPE_F32 ? 256 : 512) * p) + 16;
          most = last > most ? last : most;
        }
        if (j0 + 16 * j + i < r && at != opt_at<XT>(slots - 32 + 8 * g, j0 + 16 * j + i, rp)) ++wrong;
      }
  std::printf("%d %d %ld %ld\n", XT, r, most, wrong);
}
int main(int, char** argv) {
  const long slots = std::atol(argv[1]);
  for (int r = 1; r <= 512; ++r) {
    reach<RQ_DTYPE_F32>(r, slots);
    reach<RQ_DTYPE_BF16>(r, slots);
    reach<RQ_DTYPE_F16>(r, slots);
  }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    sys.path.insert(0, os.path.dirname(CSRC))
    import build as pkg_build
    src = tmp_path_factory.mktemp("operands") / "reach.cpp"
    src.write_text("#include <cstdlib>\n" + SOURCE)
    exe = str(src.with_suffix(""))
    subprocess.run([pkg_build.hipcc(), "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-I", CSRC, "-I", INCLUDE,
                    str(src), "-o", exe], check=True, capture_output=True, text=True)
    return exe


@pytest.mark.parametrize("M,n,grouped", [(64, 1, 0), (1, 1, 0), (32768, 1, 0), (64, 1, 1), (300, 3, 1)])
def test_row_sums_read_inside_their_operands(program, M, n, grouped):
    def u_size(r):
        b = ctypes.c_int64(0)
        nat.call("rq_multi_lora_u_size", M, n, r, grouped, ctypes.byref(b))
        return b.value
    slots = u_size(16) // 64
    out = subprocess.run([program, str(slots)], check=True, capture_output=True, text=True).stdout.split("\n")
    rows = [tuple(map(int, line.split())) for line in out if line]
    assert len(rows) == 3 * 512
    past = [(dtype, r, most - u_size(r)) for dtype, r, most, _ in rows if most > u_size(r)]
    assert not past, f"bytes past the operands' end by dtype and rank: {past[:4]} .. ({len(past)} in all)"
    assert not [row for row in rows if row[3]]
