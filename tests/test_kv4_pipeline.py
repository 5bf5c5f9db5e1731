"""The barriers of the 4-bit cache's prompt attention (k_kv4_prompt), without a
GPU: its warps as threads of a small machine whose schedule is random, so that
any of them may be stopped for any time.  A wait names a phase by its parity
only, so it must never be asked for a phase that is two behind, nor pass for
one that is still to come; and no buffer may be written while another thread
still needs it.

How many barriers a half has for P and for P V is read from the kernel's own
table of them."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tts-rs_b200", "csrc", "kv4.cu")
ROWS = 2   # softmax threads of a half (the kernel's 128, as far as barriers go)
PAGES = 2  # unpacking warps of K, and of V


def barriers_of_the_kernel():
    """(barriers of a half for p_full, for pv_done)."""
    with open(SOURCE) as f:
        text = f.read()
    at = {name: int(re.search(rf"\*{name} = bars \+ (\d+)", text).group(1)) for name in ("p_full", "pv_done", "q_full")}
    return (at["pv_done"] - at["p_full"]) // 2, (at["q_full"] - at["pv_done"]) // 2


class Fault(Exception):
    pass


class Barrier:
    def __init__(self, name, count):
        self.name, self.count, self.got, self.phase = name, count, 0, 0

    def arrive(self):
        self.got += 1
        if self.got == self.count:
            self.got, self.phase = 0, self.phase + 1

    def passed(self, n):
        """What a poll for phase n by its parity says; a fault where that is not the truth."""
        says = (self.phase & 1) != (n & 1)
        if says != (self.phase > n):
            raise Fault(f"{self.name}: a wait for phase {n} {'passes' if says else 'blocks'} at phase {self.phase}")
        return says


class Machine:
    """tiles (nt0, nt1): tiles of keys of either half; moves(h, i): whether O of half h moves at tile i."""

    def __init__(self, tiles, p_bars, pv_bars, moves):
        self.nt, self.n, self.moves = tiles, max(tiles), moves
        B = lambda name, count, n=2: [Barrier(f"{name}[{i}]", count) for i in range(n)]  # noqa: E731
        self.k_full, self.v_full = B("k_full", PAGES), B("v_full", PAGES)
        self.k_freed, self.v_freed = B("k_freed", 2), B("v_freed", 2)
        self.s_full = [B(f"s_full {h}", 2) for h in range(2)]
        self.s_freed = [B(f"s_freed {h}", ROWS) for h in range(2)]
        self.p_full = [B(f"p_full {h}", ROWS, p_bars) for h in range(2)]
        self.pv_done = [B(f"pv_done {h}", 1, pv_bars) for h in range(2)]
        # what a buffer holds: the tile, by writer
        self.k, self.v = [[None] * PAGES for _ in range(2)], [[None] * PAGES for _ in range(2)]
        self.says = [[None] * PAGES for _ in range(8)]
        self.p = [[[None] * ROWS for _ in range(2)] for _ in range(2)]
        self.s = [[None, None], [None, None]]
        self.o = [-1, -1]                # last tile that O has
        self.queues = {}                 # products and commits of an issuing thread, in order
        self.threads = {}
        for w in range(PAGES):
            self.threads[f"K{w}"] = self.unpack(w, self.k, self.k_full, self.k_freed, self.says)
            self.threads[f"V{w}"] = self.unpack(w, self.v, self.v_full, self.v_freed, None)
        for h in range(2):
            self.threads[f"S{h}"] = self.scores(h)
            self.threads[f"PV{h}"] = self.values(h)
            for r in range(ROWS):
                self.threads[f"softmax {h}.{r}"] = self.softmax(h, r)
        self.waiting = {}

    # a thread yields a condition to wait for, or None where it may be stopped
    def unpack(self, w, buf, full, freed, says):
        for i in range(self.n):
            b = i & 1
            if i >= 2:
                yield lambda b=b, n=(i >> 1) - 1: freed[b].passed(n)
            buf[b][w] = i
            if says is not None:
                says[i & 7][w] = i
            yield None
            full[b].arrive()

    def scores(self, h):
        q, other = self.queues.setdefault(f"S{h}", []), self.nt[1 - h]
        for i in range(self.nt[h]):
            b = i & 1
            yield lambda b=b, n=i >> 1: self.k_full[b].passed(n)
            if i >= 2:
                yield lambda b=b, n=(i >> 1) - 1: self.s_freed[h][b].passed(n)
            self.s_full[h][b].arrive()
            q.append(("S", h, i))
            q.append(self.s_full[h][b])
            q.append(self.k_freed[b])
            if i >= other:
                q.append(self.k_freed[b])

    def values(self, h):
        q, other = self.queues.setdefault(f"PV{h}", []), self.nt[1 - h]
        for i in range(self.nt[h]):
            b, P, D = i & 1, self.p_full[h], self.pv_done[h]
            yield lambda b=b, n=i >> 1: self.v_full[b].passed(n)
            yield lambda x=P[i % len(P)], n=i // len(P): x.passed(n)
            q.append(("PV", h, i))
            q.append(D[i % len(D)])
            q.append(self.v_freed[b])
            if i >= other:
                q.append(self.v_freed[b])

    def softmax(self, h, r):
        P, D, nt = self.p_full[h], self.pv_done[h], self.nt[h]
        done = lambda i: (lambda x=D[i % len(D)], n=i // len(D): x.passed(n))  # noqa: E731
        for i in range(nt):
            b = i & 1
            yield lambda b=b, n=i >> 1: self.s_full[h][b].passed(n)
            self.expect(self.s[h][b], i, "S")
            yield None
            for x in self.says[i & 7]:
                self.expect(x, i, "notes of K")
            self.s_freed[h][b].arrive()
            yield lambda b=b, n=i >> 1: self.v_full[b].passed(n)
            for x in self.v[b]:
                self.expect(x, i, "notes of V")
            for x in self.says[i & 7]:
                self.expect(x, i, "notes of K")
            if self.o[h] < i - 2:
                raise Fault(f"P of tile {i} is written before tile {i - 2} is in O")
            self.p[h][b][r] = i
            yield None
            if i > 0 and self.moves(h, i):
                yield done(i - 1)
                self.expect(self.o[h], i - 1, "O")
            P[i % len(P)].arrive()
        # the kernel's last waits: with one barrier for all tiles, one phase after the other
        if nt > 1 and len(D) == 1:
            yield done(nt - 2)
        if nt > 0:
            yield done(nt - 1)
            self.expect(self.o[h], nt - 1, "O")

    @staticmethod
    def expect(got, want, what):
        if got != want:
            raise Fault(f"{what}: of tile {got} instead of {want}")

    def product(self, kind, h, i):
        b = i & 1
        if kind == "S":
            for x in self.k[b]:
                self.expect(x, i, "K")
            self.s[h][b] = i
        else:
            for x in self.v[b] + self.p[h][b]:
                self.expect(x, i, "V or P")
            self.o[h] = i

    def run(self, rng, steps=20000):
        pace = {}
        for step in range(steps):
            if step % 200 == 0:  # who is slow for a while
                pace = {t: rng.choice([1, 1, 1, 0.1, 0.001]) for t in (*self.threads, *("tc " + q for q in self.queues))}
            live = [*self.threads, *("tc " + q for q, x in self.queues.items() if x)]
            if not self.threads:
                return
            t = rng.choices(live, [pace.get(x, 1) for x in live])[0]
            if t.startswith("tc "):
                item = self.queues[t[3:]].pop(0)
                item.arrive() if isinstance(item, Barrier) else self.product(*item)
                continue
            ready = self.waiting.get(t)
            if ready is not None and not ready():
                continue
            try:
                self.waiting[t] = next(self.threads[t])
            except StopIteration:
                del self.threads[t]
        raise Fault(f"not done: {sorted(self.threads)}")


def first_fault(p_bars, pv_bars, seeds):
    for seed in seeds:
        rng = random.Random(seed)
        n = rng.randint(0, 12)
        tiles = (n, rng.choice([0, n, n + rng.randint(0, 3)]) if n else rng.randint(1, 6))
        few = rng.choice([0.0, 0.1, 0.9])
        moving = {(h, i): rng.random() < few for h in range(2) for i in range(20)}
        try:
            Machine(tiles, p_bars, pv_bars, lambda h, i: moving[h, i]).run(rng)
        except Fault as f:
            return f"seed {seed}, tiles {tiles}: {f}"
    return None


def test_no_schedule_loses_a_phase_or_a_buffer():
    assert first_fault(*barriers_of_the_kernel(), range(500)) is None


@pytest.mark.parametrize("p_bars, pv_bars", [(1, 2), (2, 1)])
def test_the_machine_sees_a_barrier_that_two_tiles_share(p_bars, pv_bars):
    """One barrier of a half for all tiles: a softmax thread may arrive for a tile before another has for the one
    before it, and a second phase may be complete before the other side has asked for the first."""
    assert first_fault(p_bars, pv_bars, range(500)) is not None
