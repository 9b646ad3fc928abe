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


# ---- the barriers of the two-half form, as processes in any order -----------------------------------------------------
# Every wait of the kernel is by parity, which says what is meant only while the barrier stands in the phase that is waited
# for or just past it.  The processes below make the kernel's arrivals and waits for random units of one and two halves;
# a scheduler runs them in random order and notes each wait that passes at any other phase.

STAGES, SLOTS = 2, 4


class _Bar:
    def __init__(self, count):
        self.count, self.left, self.done = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.done = self.count, self.done + 1


def _run_protocol(units, rng, scores_first):
    bars = {}

    def bar(name, *at):
        count = 2 if name in ("KE", "VE") else 1
        return bars.setdefault((name,) + at, _Bar(count))
    wrong, pipe = [], [[], []]

    def wait(phase, name, *at):
        while (bar(name, *at).done - 1) & 1 != phase & 1:
            yield
        if bar(name, *at).done != phase + 1:
            wrong.append((name, at, phase, bar(name, *at).done))

    def loader():
        for n in range(sum(count for count, _ in units)):
            yield from wait(n // STAGES - 1, "KE", n % STAGES)
            bar("SC", n % SLOTS).arrive()
            yield
            bar("KF", n % STAGES).arrive()
            yield from wait(n // STAGES - 1, "VE", n % STAGES)
            bar("VF", n % STAGES).arrive()
            yield

    def issuer(g):
        n = k = segments = 0

        def scores(n, to):
            yield from wait(n // STAGES, "KF", n % STAGES)
            pipe[g].append([("SF", g, to), ("KE", n % STAGES)])
        for count, halves in units:
            if g < halves:
                yield from wait(segments, "QF", g)
                segments += 1
                yield from scores(n, k & 1)
                for t in range(count):
                    if t + 1 < count:
                        yield from scores(n + t + 1, (k + 1) & 1)
                    yield from wait((n + t) // STAGES, "VF", (n + t) % STAGES)
                    yield from wait(k >> 1, "PF", g, k & 1)
                    pipe[g].append([("PV", g, k & 1), ("VE", (n + t) % STAGES)])
                    k += 1
            else:
                for t in range(count):
                    yield from wait((n + t) // STAGES, "KF", (n + t) % STAGES)
                    bar("KE", (n + t) % STAGES).arrive()
                    yield from wait((n + t) // STAGES, "VF", (n + t) % STAGES)
                    bar("VE", (n + t) % STAGES).arrive()
            n += count

    def tensor(g):
        while True:
            if pipe[g]:
                for at in pipe[g].pop(0):
                    bar(*at).arrive()
            yield

    def softmax(g):
        n = done = 0
        for count, halves in units:
            if g < halves:
                bar("QF", g).arrive()
                for t in range(count):
                    k = done + t
                    waits = [("SF", k >> 1, (g, k & 1)), ("SC", (n + t) // SLOTS, ((n + t) % SLOTS,))]
                    for name, phase, at in waits if scores_first else reversed(waits):
                        yield from wait(phase, name, *at)
                    if t and rng.random() < 0.5:
                        yield from wait((k - 1) >> 1, "PV", g, (k & 1) ^ 1)
                    bar("PF", g, k & 1).arrive()
                    yield
                done += count
                yield from wait((done - 1) >> 1, "PV", g, (done - 1) & 1)
            n += count

    live = [loader(), issuer(0), issuer(1), softmax(0), softmax(1)]
    unit, steps = [tensor(0), tensor(1)], 0
    while live:
        steps += 1
        assert steps < 200000, "the processes wait for one another"
        p = rng.choice(live + unit + [live[rng.randrange(len(live))]] * rng.randrange(20))   # (some run ahead for a while)
        try:
            next(p)
        except StopIteration:
            live.remove(p)
    return wrong


def test_every_wait_finds_its_barrier_where_it_expects_it(source):
    import random
    seen = set()
    for seed in range(120):
        rng = random.Random(seed)
        units = [(rng.choice([1, 2, 3, 7, 12, 20]), rng.choice([1, 2])) for _ in range(rng.randrange(1, 8))]
        assert _run_protocol(units, rng, True) == []
        seen.update(w[0] for w in _run_protocol(units, rng, False))
    assert seen == {"SC"}                            # what the order of a tile's two waits is for
    scores, scales = (source.index("mbar_wait(bar(L::%s" % b) for b in ("B_SF", "B_SC"))
    assert scores < scales
