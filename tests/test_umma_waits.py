"""The barriers of the tcgen05 INT4 product (linear_umma.cu) as a model that
walks every interleaving of its warps, on the CPU.

A CTA's steps pass through two rings of mbarriers: `full` (the operands of a
step are written) and `empty` (its MMAs are complete).  A waiter knows a phase
by its parity alone, so it must look at every phase before the next completes,
and an arrival must not come before the phase of the ring's last turn is
complete.  The model has the warps of the two dequantising groups, those of the
activations' sums, their loader, the issuers, the MMAs' completions and the
drain; a state is how far each has come.  (The weights' ring is a plain one: its
slots and its barriers turn together.)  It looks for an MMA whose operands are
not all written, a slot overwritten before it was read, a wait that passes for
the wrong phase, and a state in which nobody can go on.
"""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-on-cpu_b200", "csrc",
                   "linear_umma.cu")


def python_of(expr):
    """A C constant expression (c ? a : b, && and !) as a Python one."""
    if "?" in expr:
        cond, rest = expr.split("?", 1)
        yes, no = rest.split(":", 1)
        return f"({python_of(yes)}) if ({python_of(cond)}) else ({python_of(no)})"
    return expr.replace("&&", " and ").replace("!", " not ").replace("/", "//").strip()


def config(fl, awq):
    """The constants of UCfg<fl, awq>, and how many entries the barrier rings have."""
    txt = open(SRC).read()
    body = re.search(r"struct UCfg \{(.*?)\n\};", txt, re.S).group(1)
    env = dict(FL=fl, AWQ=awq)
    for name, expr in re.findall(r"static constexpr (?:bool|int) (\w+) = ([^;]*);", body):
        try:
            env[name] = eval(python_of(expr), {}, env)
        except NameError:  # one that the model does not need
            pass
    full, empty = re.search(r"\bfull\[(\w+)\], empty\[(\w+)\]", txt).groups()
    return dict(a=env["kASlots"], x=env["kXSlots"], issuers=env["kAcc"], hold=env["kHold"], sums=env["kSums"],
                full=env[full], empty=env[empty])


def walk(n, a, x, issuers, hold, sums, full, empty, tma=True, warps=2, act=1):
    """What goes wrong in some interleaving of n steps, or None.

    `warps` siblings stand for a group's four, `act` for the two warps of the
    activations.  Agents that are alike are kept in order."""
    act = act if sums or not tma else 0
    group = [list(range(g, n, 2)) for g in range(2)]
    issued = [list(range(i, n, issuers)) for i in range(issuers)]
    drained = [j for j in range(n) if hold == 1 or (j // issuers + j) % hold == 0 or j + issuers >= n]
    count = warps + act
    S = 2 * warps                          # places in a state: the dequantisers, then
    P = S + act                            # the activations' warps, the loader,
    I = P + 1                              # the issuers,
    Q = I + issuers                        # their completed steps,
    R = Q + issuers                        # the drain,
    F = R + 1                              # phases of full, then what is missing to the next
    start = [0] * (F + full) + [count] * full

    def passes(phases, k):                 # a wait for phase k, where `phases` are complete
        return (phases ^ k) & 1

    def arrive(s, j):
        s[F + full + j % full] -= 1
        if s[F + full + j % full] == 0:
            s[F + full + j % full] = count
            s[F + j % full] += 1

    seen, todo = {tuple(start)}, [tuple(start)]
    while todo:
        st = todo.pop()
        complete = [st[Q + j % issuers] > j // issuers for j in range(n)]
        done = [0] * empty
        for j in range(n):
            done[j % empty] += complete[j]
        loads = [len(range(i, st[P], x)) for i in range(x)]
        out = []

        def seen_empty(j):
            """Whether a wait for step j's MMAs passes; raises where it passes too early."""
            if not passes(done[j % empty], j // empty):
                return False
            if not complete[j] or done[j % empty] != j // empty + 1:
                raise AssertionError(f"a wait for step {j} passed at another phase")
            return True

        try:
            for w in range(2 * warps):     # dequantisers: wait, then write and arrive
                g, pc = w // warps, st[w]
                if (w % warps and pc >= st[w - 1]) or pc == 2 * len(group[g]):
                    continue
                j = group[g][pc >> 1]
                s = list(st)
                s[w] += 1
                if pc & 1 == 0:
                    if j < a or seen_empty(j - a):
                        out.append(s)
                else:
                    if j >= a and not complete[j - a]:
                        raise AssertionError(f"step {j} overwrites the A slot of {j - a}")
                    arrive(s, j)
                    out.append(s)
            for w in range(act):           # sums, or plain loads of the activations
                j = st[S + w]
                if j == n or (w and st[S + w] >= st[S + w - 1]):
                    continue
                if passes(loads[j % x], j // x) if tma else j < x or seen_empty(j - x):
                    if tma and st[P] <= j:
                        raise AssertionError(f"activations of step {j} read before they landed")
                    s = list(st)
                    s[S + w] += 1
                    arrive(s, j)
                    out.append(s)
            if tma and st[P] < n and (st[P] < x or seen_empty(st[P] - x)):
                s = list(st)
                s[P] += 1
                out.append(s)
            for i in range(issuers):
                if st[I + i] < len(issued[i]):
                    j = issued[i][st[I + i]]
                    before = [k for k in issued[i][:st[I + i]] if k in drained]
                    fresh = not st[I + i] or issued[i][st[I + i] - 1] in drained
                    if (passes(st[F + j % full], j // full)
                            and (sums or not tma or passes(loads[j % x], j // x))
                            and not (fresh and before and st[R] <= drained.index(before[-1]))):
                        late = [w for w in range(warps) if st[j % 2 * warps + w] < 2 * (j // 2 + 1)]
                        if late or any(st[S + w] <= j for w in range(act)) or (tma and st[P] <= j):
                            raise AssertionError(f"the MMAs of step {j} start before its operands are written")
                        s = list(st)
                        s[I + i] += 1
                        out.append(s)
                if st[Q + i] < st[I + i]:  # its oldest MMAs complete
                    s = list(st)
                    s[Q + i] += 1
                    out.append(s)
            if st[R] < len(drained) and complete[drained[st[R]]]:
                s = list(st)
                s[R] += 1
                out.append(s)
        except AssertionError as e:
            return str(e)
        if not out and st[R] < len(drained):
            return f"nobody can go on: {st}"
        for s in out:
            t = tuple(s)
            if t not in seen:
                seen.add(t)
                todo.append(t)
    return None


KINDS = [(1, True), (2, True), (4, True), (1, False), (2, False), (4, False)]


@pytest.mark.parametrize("fl,awq", KINDS)
@pytest.mark.parametrize("tma", [True, False])
def test_every_interleaving(fl, awq, tma):
    c = config(fl, awq)
    assert walk(n=11 if c["a"] == 4 else 13, tma=tma, **c) is None


@pytest.mark.parametrize("warps,act", [(3, 1), (2, 2)])
def test_every_interleaving_of_more_siblings(warps, act):
    assert walk(n=10, warps=warps, act=act, **config(1, False)) is None


@pytest.mark.parametrize("full,empty,what", [(4, 6, "operands are written"), (6, 4, "nobody can go on")])
def test_the_model_sees_rings_that_are_too_short(full, empty, what):
    """Three A slots with barriers for four steps only: an MMA of unwritten rows,
    or a completion that a late group misses."""
    c = dict(config(1, False), full=full, empty=empty)
    assert what in (walk(n=10, **c) or "nothing")
