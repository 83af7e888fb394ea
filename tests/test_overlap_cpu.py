"""csrc/overlap.h (which calls of the policy memory's operators are refused for outputs that share memory with what they
read) against all indexes written out."""
import itertools
import os
import random
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "overlap.h"
using namespace overlap;
static bool get(Bytes& b) {
    long at, width;
    int n;
    if (std::scanf("%ld %ld %d", &at, &width, &n) != 3) return false;
    b = Bytes((const void*)at, width);
    for (int i = 0; i < n; i++) {
        long c, s;
        if (std::scanf("%ld %ld", &c, &s) != 2) return false;
        b.by(c, s);
    }
    return true;
}
int main() {
    Bytes a, b;
    while (get(a) && get(b)) std::printf("%d %d\n", (int)meet(a, b), (int)meets_itself(a));
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "ask.cpp").write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(REPO, "imitation-learning-rl_amd", "csrc"), str(d / "ask.cpp"),
                           "-o", str(d / "ask")])

    def run(pairs):
        text = "\n".join(" ".join(str(v) for piece in pair for v in (piece[0], piece[1], len(piece[2]), *itertools.chain(*piece[2])))
                         for pair in pairs)
        out = subprocess.run([str(d / "ask")], input=text, stdout=subprocess.PIPE, check=True, text=True, timeout=60).stdout
        return [tuple(int(v) for v in line.split()) for line in out.splitlines()]
    return run


def starts(piece):
    at, _, dims = piece
    return [at + sum(i * s for i, (_, s) in zip(idx, dims)) for idx in itertools.product(*[range(c) for c, _ in dims])]


def expect(a, b):
    sa, sb = starts(a), starts(b)
    both = any(x < y + b[1] and y < x + a[1] for x in sa for y in sb)
    own = any(abs(x - y) < a[1] for x, y in itertools.combinations(sa, 2))
    return int(both), int(own)


def test_small_layouts(ask):
    r = random.Random(5)

    def piece():
        dims = [(r.choice([0, 1, 2, 2, 3, 4]) if r.random() < 0.9 else 1, r.choice([-24, -8, 0, 1, 3, 4, 5, 8, 16, 20, 64])) for _ in range(r.randint(0, 3))]
        return (1000 + r.randint(-40, 40), r.randint(1, 9), dims)
    pairs = [(piece(), piece()) for _ in range(4000)]
    want = [expect(a, b) for a, b in pairs]
    assert ask(pairs) == want
    assert {w[0] for w in want} == {0, 1} == {w[1] for w in want}


def test_slices_of_packed_rows(ask):
    """Lanes of q, k, v and out side by side in one buffer, at sizes whose indexes cannot be written out."""
    lanes, steps, h, row = 1 << 19, 4096, 4, 128
    step = 4 * h * row
    lane = steps * step

    def part(i, heads=h, width=row, shift=0):
        return (1 << 40) + i * h * row + shift, width, [(lanes, lane), (steps, step), (heads, row)]
    yes, no = [], []
    for i, j in itertools.product(range(4), range(4)):
        (yes if i == j else no).append((part(i), part(j)))
    yes += [(part(0, shift=1), part(1)), (part(1, shift=-1), part(0)), (part(3, width=row + 1), part(0, shift=step)),
            (part(0), part(3, shift=2 * step + 1))]
    no += [(part(3), part(0, shift=step)), (part(3, width=row + 1), part(1)), (part(0, heads=1), part(0, shift=row, heads=3))]
    assert [x[0] for x in ask(yes)] == [1] * len(yes)
    assert [x[0] for x in ask(no)] == [0] * len(no)
    # lane-major and time-major rows inside one another's span: every step of a lane is met
    a = ((1 << 40), row, [(64, steps * row), (steps, row)])
    b = ((1 << 40) + 3 * row, row, [(64, row), (steps, 64 * row)])
    c = ((1 << 40) + 64 * steps * row, row, [(64, row), (steps, 64 * row)])
    assert [x[0] for x in ask([(a, b), (a, c), (c, b)])] == [1, 0, 1]
