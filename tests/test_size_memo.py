"""The table of per-size answers behind the launch plans (csrc/size_memo.h): however many sizes a process has seen,
each is asked for once; what could not be answered is asked for again."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <cstdio>
#include <thread>
#include <tuple>
#include <vector>
#include "size_memo.h"

struct Key {
  int dev, smem, S;
  bool operator<(const Key& o) const { return std::tie(dev, smem, S) < std::tie(o.dev, o.smem, o.S); }
};

int main() {
  fni8h::SizeMemo<Key> memo;
  int asked = 0, wrong = 0;
  for (int pass = 0; pass < 3; ++pass)
    for (int i = 0; i < 2000; ++i) {
      const Key k{i % 3, 1024 * (i / 8), 1 + i % 8};
      const int n = memo.get(k, [&] { ++asked; return k.smem + 10 * k.S + k.dev; });
      wrong += n != k.smem + 10 * k.S + k.dev;
    }
  int failed = 0;
  for (int i = 0; i < 3; ++i) wrong += memo.get(Key{9, 9, 9}, [&] { ++failed; return -1; }) != -1;
  fni8h::SizeMemo<int> shared;
  std::vector<std::thread> threads;
  int found = 0;  // counted under the table's lock
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&] { for (int i = 0; i < 500; ++i) shared.get(i, [&] { ++found; return i; }); });
  for (auto& t : threads) t.join();
  std::printf("%d %d %d %d\n", asked, wrong, failed, found);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_each_size_is_asked_for_once(tmp_path):
    src, exe = tmp_path / "memo.cpp", tmp_path / "memo"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "fni8-serve_b200", "csrc"),
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout
    assert out.split() == ["2000", "0", "3", "500"]

