"""The bounded waits of the many-row attention kernel, compiled for the host: barriers and clock are the test's."""
import os
import re
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "sageattention-rdna4_b200", "csrc", "sage_cache_tree.cu")

HOST = r"""
#include <cstdint>
#include <cstdio>
#define __device__
#define __forceinline__ inline
#define __builtin_expect(x, y) (x)
static uint32_t now, tries, complete_after, abort_word;
static int32_t host_word;
%s
struct Watch { volatile uint32_t* abort; int32_t* host; };
static uint32_t clock32() { return now; }
static bool mbar_try(uint32_t, uint32_t) { now += 1000000u; return ++tries > complete_after; }
%s
%s
int main(int argc, char**) {
  auto reset = [](uint32_t after, uint32_t aborted) { tries = 0; complete_after = after; abort_word = aborted; host_word = 0; now = 4000000000u; };
  const Watch w = {&abort_word, &host_word};
  bool ok;
  reset(50, 0); ok = mbar_wait(0, 0, w, 2); printf("%%d %%u %%u %%d\n", ok, tries, abort_word, host_word);
  reset(50, 1); ok = mbar_wait(0, 0, w, 2); printf("%%d %%u %%u %%d\n", ok, tries, abort_word, host_word);
  reset(~0u, 0); ok = mbar_wait(0, 0, w, 2); printf("%%d %%d %%u %%d\n", ok, tries < 2100, abort_word, host_word);
  reset(50, 0); drain_wait(0, w, 2); printf("%%u %%d\n", tries, host_word);
  reset(50, 1); drain_wait(0, w, 2); printf("%%u %%d\n", tries, host_word);
  reset(~0u, 1); drain_wait(0, w, 2); printf("%%d %%d\n", tries < 2100 && tries > 1900, host_word);
}
"""


def _function(text, name):
    at = re.search(r"^__device__ __forceinline__ \w+ %s\(.*?^}" % name, text, re.S | re.M)
    assert at, name
    return at.group(0)


@pytest.fixture(scope="module")
def source():
    with open(SRC) as f:
        return f.read()


def test_waits(source, tmp_path):
    limit = re.search(r"^constexpr uint32_t WAIT_CYCLES = .*?;", source, re.M).group(0)
    at = tmp_path / "waits.cc"
    at.write_text(HOST % (limit, _function(source, "mbar_wait"), _function(source, "drain_wait")))
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "waits"), str(at)], check=True)
    lines = subprocess.run([str(tmp_path / "waits")], check=True, capture_output=True, text=True).stdout.split("\n")
    assert lines[:3] == ["1 51 0 0",                 # complete after 51 tries
                         "0 2 1 0",                  # another warp has given up: this one leaves at once
                         "0 1 1 2"]                  # runs out: tells the CTA and the host
    assert lines[3:6] == ["51 0", "51 0",            # a drain waits for its products whoever has given up
                          "1 2"]                     # ... but not for good


def test_the_products_are_drained_before_their_memory_is_freed(source):
    drain, commit, free = (source.index(x) for x in ("drain_wait(bar(L::B_DRAIN)", "tc_commit(bar(L::B_DRAIN))", "tcgen05.dealloc"))
    assert commit < drain < free
    assert not re.search(r"mbar_wait\(bar\(L::B_DRAIN\)", source)
