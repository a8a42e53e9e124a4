"""Waits for barriers that end (csrc/waits.h), compiled on its own for a barrier and a clock of the test's."""
import os
import re
import subprocess

import pytest
from test_training_sources_cpu import kernels

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'ffcv_b200', 'csrc')
BEGIN = r'''
#include <stdio.h>
#include "waits.h"
using namespace ffcvb;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

static uint64_t the_time = 1000, a_try = 100; // ns, and what a try takes
static uint64_t now() { return the_time; }
// A barrier as the GPU has it: a phase's parity says whether it is over as long as the one behind it is not.
struct Barrier {
    unsigned over = 0; // phases
    bool passed(unsigned parity) {
        the_time += a_try;
        return (over & 1) != parity;
    }
};
'''
PROGRAMS = {
    # Tiles' results are in two halves in turn, each with a barrier; those of `made` tiles are there, and no more will be.
    'a waiter that has given up takes nothing': r'''
int main() {
    for (int made = 0; made < 9; made++) {
        Barrier done[2];
        volatile int gave_up = 0;
        Waiter waiter(&gave_up);
        bool stale = false;
        for (int m = 0; m < 20; m++) {
            if (m < made) done[m & 1].over++;
            const unsigned parity = m / 2 & 1;
            const bool fine = waiter([&] { return done[m & 1].passed(parity); }, now);
            CHECK(fine == (m < made) && waiter.fine == fine && (gave_up != 0) == !fine);
            Waiter another(&gave_up); // one that does not know what has been missed
            stale |= m > made && another([&] { return done[m & 1].passed(parity); }, now);
        }
        CHECK(stale);
    }
    return 0;
}
''',
    'a wait ends': r'''
int main() {
    Barrier done;
    for (uint64_t each = 100; each <= 1000000; each *= 10) {
        a_try = each;
        volatile int gave_up = 0;
        Waiter one(&gave_up), other(&gave_up);
        uint64_t before = the_time;
        CHECK(!one([&] { return done.passed(0); }, now) && gave_up == 1);
        CHECK(the_time - before >= kLongestWait && the_time - before <= kLongestWait + 200 * a_try);
        before = the_time;
        CHECK(!other([&] { return done.passed(0); }, now) && the_time - before <= 70 * a_try); // (another one is told)
        CHECK(!one([&] { return true; }, now));
        Waiter lucky(&gave_up); // what is there is taken all the same
        done.over++;
        CHECK(lucky([&] { return done.passed(0); }, now) && lucky.fine);
        done.over++;
    }
    return 0;
}
''',
    'time off the GPU is not waited': r'''
int main() {
    for (int tries = 0; tries < 3000; tries += 7) { // (the block is off the GPU for an hour, after so many tries)
        Barrier done;
        volatile int gave_up = 0;
        Waiter waiter(&gave_up);
        a_try = 100;
        int left = tries;
        const bool fine = waiter([&] {
            if (left-- == 0) the_time += 3600000000000ull;
            if (left == -1000) done.over++;
            return done.passed(0);
        }, now);
        CHECK(fine && !gave_up);
    }
    // but one that is on and off again and again does not wait for good
    Barrier never;
    volatile int gave_up = 0;
    Waiter waiter(&gave_up);
    int tries = 0;
    CHECK(!waiter([&] { tries++, the_time += 3600000000000ull; return never.passed(0); }, now) && tries <= 64 * 23);
    return 0;
}
''',
}


@pytest.mark.parametrize('what', PROGRAMS)
def test_waits(what, tmp_path):
    source, program = tmp_path / 'waits.cpp', tmp_path / 'waits'
    source.write_text(BEGIN + PROGRAMS[what])
    subprocess.run(['g++', '-std=c++17', '-O2', '-Wall', '-Werror', '-I', CSRC, '-o', str(program), str(source)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout


def products_kernel():
    body, = (body for _, body in kernels('linear_cross_entropy.cu') if 'multiply<' in body)
    return body


def test_who_has_given_up_gives_nothing_back():
    """A half of the results is multiplied over once eight warps have arrived for it: arrivals for tiles that a warp has not waited for would stand for those
    of warps that still read theirs."""
    give_back = re.search(r'auto give_back = \[&\] \{(.*?)\n {12}\};', products_kernel(), re.S).group(1)
    assert give_back.index('|| !fine) return;') < give_back.index('barrier_arrive')


def test_copies_are_waited_for_whoever_has_given_up():
    """A block that ends has no copy on its way, even if all were issued before others gave up: its shared memory is another's then.  (Those of a pair whose stages have
    all been freed have been multiplied.)"""
    copying = products_kernel().split('} else if (warp == 1) {')[0]
    last = re.search(r'\n {12}if \(rank == 0 && !\(PAIR && fine\)\)[^\n]*\n(.*?)\n {12}\S', copying + '\n            .', re.S).group(1)
    assert 'patient(&mine)' in last and 'barrier_wait(patient, full' in last
    assert copying.index('for (Walk<MODE> walk') < copying.index('barrier_wait(waiter, empty + 8 * (k') < copying.index('barrier_wait(patient, full')
