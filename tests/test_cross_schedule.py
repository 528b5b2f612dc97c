"""CPU replay of the cross-attention kernels' barriers (``csrc/cross_attn.cu``,
``csrc/cross_attn_bwd.cu``).

Every role of a CTA is a generator of waits and arrivals in its kernel's order;
loads and matrix instructions complete later, in the order in which their role
issued them.  A wait knows one parity bit only, as on the GPU: it passes when the
barrier's unfinished phase has the other parity.  Whatever the order in which the
roles run (drawn at random, or with one role held back until nothing else can
move), a wait has to pass in the phase that it was meant for: not in an earlier
one, and not be found two phases behind, where it would read "not yet" until the
kernel's limit ends the call."""

import random

import pytest


class Violation(AssertionError):
    pass


class Barriers:
    def __init__(self, counts):
        self.counts, self.done, self.left = counts, {}, {}

    def arrive(self, bar):
        count = self.counts.get(bar[0], 1)
        left = self.left.get(bar, count) - 1
        if left == 0:
            self.done[bar] = self.done.get(bar, 0) + 1
            left = count
        self.left[bar] = left

    def passes(self, role, bar, phase):
        done = self.done.get(bar, 0)  # phases completed: the unfinished one has this number
        if (done & 1) != (phase & 1):
            if done != phase + 1:
                raise Violation(f"{role}: phase {phase} of {bar} passed after {done} phases")
            return True
        if done > phase:
            raise Violation(f"{role}: phase {phase} of {bar} missed, {done} phases are over")
        return False


def replay(roles, counts, rng, held=None, after=0):
    """Run ``{name: generator}`` to the end: one step of a role or one completion at a time.
    ``held``: the role that, after so many steps of its own, moves only when nothing else can."""
    bars = Barriers(counts)
    waiting = {name: next(gen, None) for name, gen in roles.items()}
    later = {name: [] for name in roles}
    while True:
        ready = [("done", n) for n, q in later.items() if q]
        for n, act in waiting.items():
            if act is not None and (act[0] != "wait" or bars.passes(n, act[1], act[2])):
                ready.append(("step", n))
        if not ready:
            break
        others = [r for r in ready if after > 0 or r != ("step", held)]
        kind, n = rng.choice(others or ready)
        if kind == "done":
            bars.arrive(later[n].pop(0))
            continue
        act = waiting[n]
        if act[0] == "arrive":
            bars.arrive(act[1])
        elif act[0] == "later":
            later[n].append(act[1])
        waiting[n] = next(roles[n], None)
        after -= n == held
    stuck = {n: a for n, a in waiting.items() if a is not None}
    if stuck:
        raise Violation(f"stuck: {stuck}")


# A role yields ("wait", barrier, phase), ("arrive", barrier) or ("later", barrier): the arrival of a
# load or of a commit behind the matrix instructions issued so far.


def wait(name, i, phase):
    return ("wait", (name, i), phase)


def arrive(name, i=0):
    return ("arrive", (name, i))


def later(name, i=0):
    return ("later", (name, i))


def steps(items):
    """``(j, i, u, cnt)`` of the steps of the items that have any: item, step of the item, step of the CTA."""
    u = 0
    for j, cnt in enumerate(c for c in items if c):
        for i in range(cnt):
            yield j, i, u, cnt
            u += 1


def dq_kernel(items, one_step_waits=True):
    """``cross_bwd_dq_tcgen05``; ``one_step_waits`` false leaves out the wait for the delta warps
    where an item is one step long."""

    def query_tiles():
        n = sum(1 for c in items if c)
        for j in range(n):
            if j >= 2:
                yield wait("TE", j % 2, j // 2 - 1)
            yield later("TF", j % 2)
        for j in range(max(0, n - 2), n):
            yield wait("TE", j % 2, j // 2)

    def keys():
        for _, _, u, _ in steps(items):
            yield wait("KE", u % 4, u // 4 - 1)
            yield later("KF", u % 4)
            yield wait("VE", u % 2, u // 2 - 1)
            yield later("VF", u % 2)

    def scores():
        for j, i, u, _ in steps(items):
            if i == 0:
                yield wait("TF", j % 2, j // 2)
            yield wait("KF", u % 4, u // 4)
            yield wait("VF", u % 2, u // 2)
            yield wait("DQ", u % 3, u // 3 - 1)
            yield later("SF", u % 3)
            yield later("VE", u % 2)

    def gradient():
        for j, i, u, _ in steps(items):
            yield wait("DS", u % 3, u // 3)
            if i == 0:
                yield wait("OE", 0, j - 1)
            yield later("DQ", u % 3)
            yield later("KE", u % 4)

    def delta():
        for j, i, _, _ in steps(items):
            if i == 0:
                yield wait("TF", j % 2, j // 2)
                yield arrive("DR", j % 2)

    def softmax(g):
        have = -1
        for j, i, u, cnt in steps(items):
            if u % 3 != g:
                continue
            yield wait("SF", g, u // 3)
            if have != j and (cnt > 1 or one_step_waits):
                yield wait("DR", j % 2, j // 2)
            have = j
            yield arrive("DS", g)
            if i + 1 == cnt:
                yield wait("DQ", g, u // 3)
                yield arrive("OE")
                yield arrive("TE", j % 2)

    roles = {"query tiles": query_tiles(), "keys": keys(), "scores": scores(), "gradient": gradient()}
    roles.update({f"delta warp {w}": delta() for w in range(4)})
    roles.update({f"softmax {g} warp {w}": softmax(g) for g in range(3) for w in range(4)})
    return roles, dict.fromkeys(("DR", "DS", "OE", "TE"), 4)


def dkdv_kernel(segments):
    """``cross_bwd_dkdv_tcgen05``: segments of so many steps each."""
    run = [(s, i, r, n) for r, (s, i, n) in enumerate((s, i, n) for s, n in enumerate(segments) for i in range(n))]

    def loads():
        for s, i, r, _ in run:
            if i == 0:
                if s > 0:
                    yield wait("AF", 0, s - 1)
                yield later("TF")
            yield wait("RE", r % 4, r // 4 - 1)
            yield later("RF", r % 4)

    def products():
        for s, i, r, n in run:
            if i == 0:
                yield wait("TF", 0, s)
            yield wait("RF", r % 4, r // 4)
            yield later("SF", r % 2)
            if i == 0:
                yield wait("AE", 0, s - 1)
            else:
                yield wait("DS", (r - 1) % 2, (r - 1) // 2)
                yield later("RE", (r - 1) % 4)
            if i + 1 == n:
                yield wait("DS", r % 2, r // 2)
                yield later("RE", r % 4)
                yield later("AF")

    def softmax():
        for s, i, r, n in run:
            yield wait("RF", r % 4, r // 4)
            yield wait("SF", r % 2, r // 2)
            yield arrive("DS", r % 2)
            if i + 1 == n:
                yield wait("AF", 0, s)
                yield arrive("AE")

    roles = {"loads": loads(), "products": products()}
    roles.update({f"softmax warp {w}": softmax() for w in range(8)})
    return roles, {"DS": 8, "AE": 8}


def forward_kernel(items, rescale):
    """``cross_attn_tcgen05`` without slices; ``rescale(u)``: whether unit u rescales O."""

    def in_q(cnt):
        return cnt >= 3

    def query_tiles():
        held, uses, k = {}, {0: 0, 1: 0}, 0
        j = 0
        for cnt in items:
            if cnt == 0:
                continue
            e = j % 2
            yield wait("QE", e, j // 2 - 1)
            if held.pop(e, False):
                yield wait("OQ", e, uses[e] - 1)
            if in_q(cnt):
                held[e] = True
                uses[e] += 1
            yield later("QF", e)
            for _ in range(cnt):
                yield wait("KE", k % 2, k // 2 - 1)
                yield later("KF", k % 2)
                k += 1
            j += 1
        for e in (j % 2, (j + 1) % 2):
            if held.pop(e, False):
                yield wait("OQ", e, uses[e] - 1)

    def values():
        held, uses = {}, {0: 0, 1: 0, 2: 0}
        last = 0
        for _, i, u, cnt in steps(items):
            f = u % 3
            yield wait("VE", f, u // 3 - 1)
            if held.pop(f, False):
                yield wait("OV", f, uses[f] - 1)
            yield later("VF", f)
            if i + 1 == cnt and not in_q(cnt):
                held[f] = True
                uses[f] += 1
            last = u
        for n in range(1, 4):
            if held.pop((last + n) % 3, False):
                yield wait("OV", (last + n) % 3, uses[(last + n) % 3] - 1)

    def scores():
        for j, i, u, cnt in steps(items):
            if i == 0:
                yield wait("QF", j % 2, j // 2)
            yield wait("KF", u % 2, u // 2)
            yield wait("PV", u % 3, u // 3 - 1)
            yield later("SF", u % 3)
            yield later("KE", u % 2)
            if i + 1 == cnt:
                yield later("QE", j % 2)

    def outputs():
        for j, i, u, _ in steps(items):
            yield wait("VF", u % 3, u // 3)
            if i == 0:
                yield wait("OE", 0, j - 1)
            yield wait("PB", u % 3, u // 3)
            yield wait("PA", u % 3, u // 3)
            yield later("VE", u % 3)
            yield later("PV", u % 3)

    def softmax(g):
        for j, i, u, cnt in steps(items):
            if u % 3 != g:
                continue
            yield wait("SF", g, u // 3)
            if u > 0:
                yield wait("MR", (u - 1) % 3, (u - 1) // 3)
            yield arrive("MR", g)
            if i > 0 and rescale(u):
                yield wait("PV", (u - 1) % 3, (u - 1) // 3)
            yield arrive("PB", g)
            yield arrive("PA", g)
            if u > 0:
                yield wait("LR", (u - 1) % 3, (u - 1) // 3)
            yield arrive("LR", g)
            if i + 1 == cnt:
                yield wait("PV", g, u // 3)
                yield arrive("OE")
                yield arrive("OQ", j % 2) if in_q(cnt) else arrive("OV", u % 3)

    roles = {"query tiles": query_tiles(), "values": values(), "scores": scores(), "outputs": outputs()}
    roles.update({f"softmax {g} warp {w}": softmax(g) for g in range(3) for w in range(4)})
    return roles, dict.fromkeys(("PA", "PB", "MR", "LR", "OE", "OQ", "OV"), 4)


# steps of the items of a CTA: of one step, of one and of several by turns (lengths of a batch), without keys
ITEMS = {
    "one_step": [1] * 9,
    "two_steps": [2] * 6,
    "one_then_many": [1, 1, 4, 1, 5, 1, 1, 1, 3],
    "empty_between": [0, 1, 0, 0, 3, 1, 0, 1, 2, 0],
    "long": [9, 8],
    "single": [1],
}


def _orders(make, seeds=12):
    """Every role held back in turn, from its start and from each of its first steps, then random orders."""
    for held in make()[0]:
        for after in range(6):
            roles, counts = make()
            replay(roles, counts, random.Random(f"{held} {after}"), held, after)
    for seed in range(seeds):
        roles, counts = make()
        replay(roles, counts, random.Random(seed))


@pytest.mark.parametrize("items", sorted(ITEMS))
def test_dq_kernel_waits_for_the_right_phase(items):
    _orders(lambda: dq_kernel(ITEMS[items]))


@pytest.mark.parametrize("items, found", [("one_step", "missed"), ("one_then_many", "missed|passed")])
def test_dq_kernel_without_the_wait_of_one_step_items(items, found):
    """Held back, a delta warp loses its place: nothing keeps the tile's reload behind it."""
    with pytest.raises(Violation, match=found):
        _orders(lambda: dq_kernel(ITEMS[items], one_step_waits=False))


def test_dq_kernel_without_the_wait_reads_an_older_delta():
    """The other side of the same missing wait: with a delta warp late between its item's load and its
    arrival, an item of several steps passes on the phase of the one-step item before it in its slot."""
    with pytest.raises(Violation, match=r"softmax \d warp \d: phase 1 of \('DR', 0\) passed after 0 phases"):
        for seed in range(1000):
            roles, counts = dq_kernel([1, 1, 2], one_step_waits=False)
            replay(roles, counts, random.Random(seed), "delta warp 2", after=1)


@pytest.mark.parametrize("segments", [[1], [1, 1, 1, 1], [5, 1, 2, 7], [12], [2, 1, 1, 3, 4]])
def test_dkdv_kernel_waits_for_the_right_phase(segments):
    _orders(lambda: dkdv_kernel(segments))


@pytest.mark.parametrize("rescale", ["never", "always", "some"])
@pytest.mark.parametrize("items", sorted(ITEMS))
def test_forward_kernel_waits_for_the_right_phase(items, rescale):
    pick = {"never": lambda u: False, "always": lambda u: True, "some": lambda u: u * 7 % 3 == 1}[rescale]
    _orders(lambda: forward_kernel(ITEMS[items], pick))
