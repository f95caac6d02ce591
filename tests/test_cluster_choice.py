"""The rules that divide an item over a cluster's blocks, on devices that do not hold every cluster size (host code alone, no GPU)."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "asrq_b200", "csrc")

PROGRAM = r"""
#include "cluster_choice.h"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
using namespace asrq;
int main(int argc, char** argv) {  // largest cluster the device holds; whether a query fails where it does not
  const int largest = atoi(argv[1]), no_answer = atoi(argv[2]);
  auto slots = [&](int split, int warps) {
    const int a_SM = 16 / warps < 1 ? 1 : 16 / warps;
    return slots_held(split <= largest ? 148 / split * a_SM : no_answer ? -1 : 0, split, 148);
  };
  for (unsigned items : {1u, 20u, 40u, 320u, 5000u})
    for (unsigned chunks : {0u, 1u, 47u, 500u, 100000u}) {
      const RowsChoice c = choose_rows(items, chunks, slots);
      printf("rows %d %d\n", c.split, c.warps);
    }
  for (int b : {1, 2, 9, 18, 40, 64, 200}) printf("select %d\n", choose_select(b, 148, largest >= 16, [](int n) { return n >= 4; }));
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("choice")
    (at / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(at / "main.cpp"), "-o", str(at / "main")], check=True)
    return str(at / "main")


@pytest.mark.parametrize("largest", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("no_answer", [0, 1])
def test_only_clusters_that_the_device_holds(program, largest, no_answer):
    lines = subprocess.run([program, str(largest), str(no_answer)], check=True, capture_output=True, text=True).stdout.split("\n")
    rows = [tuple(map(int, x.split()[1:])) for x in lines if x.startswith("rows")]
    assert len(rows) == 25 and all(1 <= s <= largest and 1 <= w <= 8 for s, w in rows)
    assert largest == 1 or any(s > 1 for s, _ in rows)
    select = [int(x.split()[1]) for x in lines if x.startswith("select")]
    assert len(select) == 7 and all(2 <= n <= (16 if largest >= 16 else 8) for n in select) and select[0] == (16 if largest >= 16 else 8)
    assert min(select) == 4  # not below what the segments' lists take
