"""Records of given-up waits (csrc/wait_record.h), on the CPU with words that the
test writes: a record stays with its device, and every thread that uses the
device learns of it once, whichever polls first."""
import os
import subprocess

from conftest import ROOT

TEST = r"""
#include <cstdio>
#include <thread>
#include "wait_record.h"

static int words[mx::WaitRecords::kDevices];
static mx::WaitRecords records(words);
static int bad = 0;
#define EXPECT(a, b) do { int x = (a), y = (b); if (x != y) ++bad, printf("line %d: %d, not %d\n", __LINE__, x, y); } while (0)

int main() {
  EXPECT(records.pending(0), 0);
  EXPECT(records.take(0), 0);
  // A record: refused until polled, told once, and only on its device.
  words[0] = 0x203;
  EXPECT(records.pending(1), 0);
  EXPECT(records.take(1), 0);
  EXPECT(records.pending(0), 0x203);
  EXPECT(records.pending(0), 0x203);
  EXPECT(records.take(0), 0x203);
  EXPECT(records.pending(0), 0);
  EXPECT(records.take(0), 0);
  // Two threads that both use the device: the one's poll does not clear the other's.
  std::atomic<int> step{0};
  auto await = [&](int s) { while (step != s) std::this_thread::yield(); };
  std::thread other([&] {
    EXPECT(records.pending(0), 0);  // what was taken before its first call
    step = 1;
    await(2);
    EXPECT(records.pending(0), 0x204);
    EXPECT(records.take(0), 0x204);
    EXPECT(records.take(0), 0);
    step = 3;
  });
  await(1);
  words[0] = 0x204;
  EXPECT(records.take(0), 0x204);
  EXPECT(words[0], 0);
  step = 2;
  await(3);
  other.join();
  EXPECT(records.pending(0), 0);
  // A second record after the first was taken, and two before anyone looked.
  words[0] = 0x201;
  EXPECT(records.take(0), 0x201);
  words[0] = 0x201;
  EXPECT(records.pending(0), 0x201);
  words[0] = 0x205;
  EXPECT(records.take(0), 0x205);
  EXPECT(records.take(0), 0);
  // A thread whose first call finds a record that nobody has seen is told of it.
  words[2] = 0x202;
  std::thread late([&] { EXPECT(records.pending(2), 0x202); });
  late.join();
  // And so is one that had used the device before.
  words[3] = 0;
  EXPECT(records.pending(3), 0);
  words[3] = 0x205;
  std::thread first([&] { EXPECT(records.take(3), 0x205); });
  first.join();
  EXPECT(records.pending(3), 0x205);
  return bad != 0;
}
"""


def test_every_thread_is_told_once(tmp_path):
    src = tmp_path / "records.cpp"
    src.write_text(TEST)
    exe = tmp_path / "records"
    subprocess.run(["g++", "-O1", "-std=c++17", "-pthread", "-I", os.path.join(ROOT, "maxim-rs_b200", "csrc"), str(src),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
