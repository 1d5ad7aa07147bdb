"""CPU: the code and message that a handle's status call makes of the words its kernels set."""
import os
import subprocess

import pytest

from conftest import ROOT

MAIN = r"""
#include <cstdio>
#include "status.h"
int main() {
  for (int bad = 0; bad < 2; ++bad)
    for (int late = 0; late < 2; ++late) {
      int words[lc::kStatusBits] = {};
      words[lc::kBadInput] = bad;
      words[lc::kTimedOut] = late;
      const int code = lc::status_code(words);
      std::printf("%d %d %d %s\n", bad, late, code, lc::status_message(code));
    }
}
"""


def test_status_words(lc, tmp_path):
    src, exe = tmp_path / "main.cpp", tmp_path / "main"
    src.write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "lumen-rs_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    lines = [x.split(" ", 3) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()]
    told = {(x[0], x[1]): (int(x[2]), x[3] if len(x) > 3 else "") for x in lines}
    assert told["0", "0"] == (lc.LC_OK, "")
    assert told["1", "0"][0] == lc.LC_ERR_INVALID and "page" in told["1", "0"][1]
    # a copy that did not come is told as that, whatever else was met
    for key in (("0", "1"), ("1", "1")):
        assert told[key][0] == lc.LC_ERR_TIMEOUT and "time" in told[key][1]


@pytest.mark.gpu
def test_status_of_a_good_call(lc, gpu):
    import torch

    beam = lc.BeamSearch(1, 2, 100)
    beam.select(torch.zeros((1, 2, 100), device="cuda"), torch.zeros((1, 2), device="cuda"))
    torch.cuda.synchronize()
    assert beam.status() == lc.LC_OK
    assert lc.lib().lc_beam_status(None) == lc.LC_ERR_INVALID
