"""CPU model of how a CTA pair of the int8 tensor-core kernel that gives up waits for its copies: two producers fill the
stages of one ring, the leader's barriers count the bytes of both, and each part stops wherever a wait of its own ran
out.  Whatever the interleaving, the waits must end, and not before every byte asked for has landed."""
import random

import pytest

WEIGHTS, TOKENS = 16384, 4096


class Barrier:
    """One arrival and the expected bytes complete a phase."""

    def __init__(self):
        self.phase, self.pending, self.bytes = 0, 1, 0

    def check(self):
        if self.pending == 0 and self.bytes == 0:
            self.phase, self.pending = self.phase + 1, 1

    def expect(self, n):
        assert self.pending == 1, "armed twice in a phase"
        self.bytes += n
        self.pending = 0
        self.check()

    def complete(self, n):
        self.bytes -= n
        self.check()


def blocks(f, sub, kblocks, wide):
    per_tile = (kblocks + sub - 1) // sub
    return sub if wide else min(sub, kblocks - (f % per_tile) * sub)


def run(seed):
    rng = random.Random(seed)
    stages, sub, kblocks = rng.randint(2, 12), rng.randint(1, 4), rng.randint(1, 40)
    wide, fills = rng.random() < 0.5, rng.randint(1, 60)
    full = [Barrier() for _ in range(stages)]
    flying, missing = [], {}          # copies under way; bytes of fill f that have not landed

    def size(f):
        b = blocks(f, sub, kblocks, wide)
        return b * WEIGHTS, b * TOKENS

    def ask(f, n):
        flying.append((f, n))
        missing[f] = missing.get(f, 0) + n

    def land():
        f, n = flying.pop(rng.randrange(len(flying)))
        missing[f] -= n
        full[f % stages].complete(n)

    def weights(r, f):
        if r == 0:
            full[f % stages].expect(2 * sum(size(f)))
        ask(f, size(f)[0])

    first_tile = (kblocks + sub - 1) // sub
    early = [rng.choice([0, min(stages, first_tile, fills)])] * 2      # weights of the first tile, ahead of the quantizer
    early = [min(n, rng.choice([n, rng.randint(0, n)])) for n in early]
    for r in (0, 1):
        for f in range(early[r]):
            weights(r, f)
    done, used = [0, 0], 0            # fills of each producer, stages that the issuer has multiplied
    stop = [rng.randint(0, fills), rng.randint(0, fills), rng.randint(0, fills)]
    for _ in range(2000):
        what = rng.randrange(4)
        if what == 3:
            if flying:
                land()
        elif what == 2:
            if used < min(stop[2], fills) and full[used % stages].phase > used // stages:
                used += 1
        elif done[what] < stop[what] and (done[what] < stages or done[what] - stages < used):
            f = done[what]
            if f >= early[what]:
                weights(what, f)
            ask(f, size(f)[1])
            done[what] += 1

    # what the leader does behind the closing barrier
    f0, f1 = done
    w0, w1 = max(f0, early[0]), max(f1, early[1])
    end = max(w0, w1)
    for f in range(max(0, end - stages), end):
        w, t = size(f)
        bar = full[f % stages]
        never = (w if f >= w0 else 0) + (t if f >= f0 else 0) + (w if f >= w1 else 0) + (t if f >= f1 else 0)
        if f >= w0:
            bar.expect(2 * (w + t))
        if never:
            bar.complete(never)
        while bar.phase <= f // stages:
            assert flying, "a wait that nothing ends"
            land()
        assert missing.get(f, 0) == 0, "the wait ended before its copies"
    assert not flying and not any(missing.values())


@pytest.mark.parametrize("start", range(0, 4000, 1000))
def test_every_copy_is_waited_for(start):
    for seed in range(start, start + 1000):
        run(seed)
