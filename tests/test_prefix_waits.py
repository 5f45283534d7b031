"""The waits of the prefix pass (prefix_attn_kernel), tried in every order that
its actors can run in.

The pass has no lock step: the MMA warp issues S(0), S(1), PV(0), S(2), PV(1),
...; the tensor core works them off in that order; each pair of softmax warps
takes S(j), writes P(j) and goes on by itself.  They meet at mbarriers, whose
wait names a parity: it passes when the phase in progress has the other parity,
so it cannot tell phase k from phase k - 2.  A wait is right only where the
waiter cannot be two phases away.  Here each actor is a generator of the waits
and arrivals that the kernel makes, and all interleavings are searched for one
in which a wait passes before what it stands for has happened."""
import pytest


def phase(k):
    """(barrier of the pair, parity) of step k on barriers kept for even and for odd steps."""
    return k & 1, (k >> 1) & 1


class Waits:
    """The kernel's: PV(k) is known by p_free, which each softmax warp follows phase by phase."""

    @staticmethod
    def pv(k):
        b, parity = phase(k)
        return ("p_free", b), parity


class OneBarrier(Waits):
    """A single barrier that every PV completes: not followed phase by phase."""

    @staticmethod
    def pv(k):
        return ("pv_done", 0), k & 1


def mma(n):
    for j in range(min(2, n)):
        yield "issue", ("S", j)
    for j in range(n):
        b, parity = phase(j)
        yield "wait", (("p_full", b), parity, None)
        yield "issue", ("PV", j)
        if j + 2 < n:
            yield "wait", (("s_free", b), parity, None)
            yield "issue", ("S", j + 2)


def softmax(n, rescales, rule):
    for j in range(n):
        b, parity = phase(j)
        yield "wait", (("s_full", b), parity, ("S", j))
        yield "arrive", ("s_free", b)
        if j >= 2:
            yield "wait", (("p_free", b), phase(j - 2)[1], ("PV", j - 2))  # P's buffer is read no more
        if j in rescales:
            bar, parity1 = rule.pv(j - 1)
            yield "wait", (bar, parity1, ("PV", j - 1))  # O is at rest
        yield "arrive", ("p_full", b)
    bar, parity = rule.pv(n - 1)
    yield "wait", (bar, parity, ("PV", n - 1))  # O is whole, P's buffers are free


def search(n, rescales, rule):
    """The first wait that passes early, or None.  rescales: per softmax pair, its steps."""
    programs = [list(mma(n))] + [list(softmax(n, r, rule)) for r in rescales]
    need = {"p_full": len(rescales), "s_free": len(rescales)}  # arrivals of a phase (others: one)
    names = ("s_full", "s_free", "p_full", "p_free", "pv_done")
    index = {(name, b): i for i, (name, b) in enumerate((name, b) for name in names for b in (0, 1))}
    start = (tuple(0 for _ in programs), 0, (), tuple((0, 0) for _ in index))
    order = [("S", 0), ("S", 1)][: min(2, n)]  # issue order
    for j in range(n):
        order.append(("PV", j))
        if j + 2 < n:
            order.append(("S", j + 2))

    def arrive(bars, bar):
        i = index[bar]
        phases, count = bars[i]
        full = count + 1 == need.get(bar[0], 1)
        return bars[:i] + (((phases + 1, 0) if full else (phases, count + 1)),) + bars[i + 1:]

    seen, todo, ended = {start}, [start], False
    while todo:
        at, done, pending, bars = todo.pop()
        issued = sum(1 for kind, _ in programs[0][: at[0]] if kind == "issue")
        after = []
        if done < issued:  # the tensor core finishes the next operation; its commits arrive in any order
            op, j = order[done]
            arrivals = (("s_full", j & 1),) if op == "S" else (("p_free", j & 1), ("pv_done", 0))
            after.append((at, done + 1, pending + arrivals, bars))
        for i, bar in enumerate(pending):
            after.append((at, done, pending[:i] + pending[i + 1:], arrive(bars, bar)))
        for w, prog in enumerate(programs):
            if at[w] == len(prog):
                continue
            kind, arg = prog[at[w]]
            step = at[:w] + (at[w] + 1,) + at[w + 1:]
            if kind == "wait":
                bar, parity, stands_for = arg
                if bars[index[bar]][0] & 1 == parity:
                    continue  # the phase of this parity is in progress
                if stands_for and stands_for not in order[:done]:
                    return w, at[w], stands_for
                after.append((step, done, pending, bars))
            elif kind == "arrive":
                after.append((step, done, pending, arrive(bars, arg)))
            else:
                after.append((step, done, pending, bars))
        if not after:
            assert all(a == len(p) for a, p in zip(at, programs)), "an actor waits for good"
            ended = True
        for state in after:
            if state not in seen:
                seen.add(state)
                todo.append(state)
    assert ended
    return None


RESCALES = [((), ()), ((1,), ()), ((2, 3), (1,)), ((1, 2, 3, 4), ()), ((4,), (3,))]


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("rescales", RESCALES)
def test_no_wait_passes_early(n, rescales):
    assert search(n, rescales, Waits) is None


def test_one_barrier_for_every_product_passes_early():
    """Why PV(k) has no barrier of its own for all k: from two steps on, a pair that
    is ahead passes the last wait while the product before the last is still pending."""
    assert search(1, ((), ()), OneBarrier) is None
    for n in (2, 3, 4):
        _, _, missing = search(n, ((), ()), OneBarrier)
        assert missing == ("PV", n - 1)
