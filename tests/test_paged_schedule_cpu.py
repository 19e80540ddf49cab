"""The barriers of the paged attention kernel, over many units of work a block, run on the CPU against each other.

The kernel's own source is compiled for the host and printed by representative threads (``host_paged``): what each waits for,
arrives on, loads, issues and touches, unit after unit.  The printed programs of the producer, the two issuers, the warp that
describes units and the warps of both softmax groups are then run against each other in many orders: each of them in turn as
late and as early as it can be, and at random.  Loads land in any order, MMAs and commits run in the order of their issuer at
any time after it has issued them, and an mbarrier is its phase, the arrivals that the phase still waits for and its outstanding
copies, so that a parity wait can pass a phase early, or block for ever, as the real one does.

One run says which write each access to Q, a slot of the K/V ring, S, P or O follows; in all others it has to follow the same, and
all have to end.  Mistakes planted in a copy of the source have to be found."""
import functools
import itertools
import os
import random
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "diffusers-tpu_b200", "csrc")
SOURCE = "paged_attn.cuh"


class Wrong(Exception):
    pass


# ---------------------------------------------------------------------------------------------------------------- programs
def _without_asm(text):
    """Inline assembly goes: what matters of it has stand-ins."""
    out, at = [], 0
    for m in re.finditer(r"\basm\b(\s+volatile)?\s*\(", text):
        if m.start() < at:
            continue
        depth, quoted, i = 1, False, m.end()
        while depth:
            if text[i] == '"':
                quoted = not quoted
            elif not quoted:
                depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        out.append(text[at:m.start()])
        at = i
    return "".join(out) + text[at:]


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """edits -> path of the tracing program, with the edits ((old, new), ...) made in a copy of the source."""
    @functools.cache
    def build(edits=()):
        folder = tmp_path_factory.mktemp("trace")
        for path, name in ((os.path.join(HERE, "host_trace", "ptx.cuh"), "trace_ptx.cuh"), (os.path.join(HERE, "host_paged", "ptx.cuh"), "ptx.cuh"),
                           (os.path.join(HERE, "host_paged", "trace.cc"), "trace.cc"), *((os.path.join(CSRC, n), n) for n in ("paged.cuh", "paged_plan.cuh", SOURCE))):
            with open(path) as f:
                text = f.read()
            if name == SOURCE:
                for old, new in (("make_plan(p.plan, scratch, blocks, me)", "host_plan(scratch)"), ("#include <cuda_fp16.h>", ""), *edits):
                    assert text.count(old) == 1, f"{old!r} stands {text.count(old)} times in {name}"
                    text = text.replace(old, new)
                begin = text.index("__device__ __forceinline__ void tmem_ld16_sync")
                text = _without_asm(text[:begin] + text[text.index("\n}\n", begin) + 3:])
            (folder / name).write_text(text)
        subprocess.run(["g++", "-std=c++17", "-O0", "-w", "-I", str(folder), str(folder / "trace.cc"), "-o", str(folder / "trace")],
                       check=True, capture_output=True, text=True)
        return str(folder / "trace")

    return build


def _trace(program, D, kernel, mode, G, warps, units):
    text = subprocess.run([program, str(D), kernel, mode, str(G), str(warps), *(f"{n}:{kv}" for n, kv in units)], check=True, capture_output=True,
                          text=True).stdout
    roles, names, counts, events = {}, {}, {}, None
    for line in text.splitlines():
        kind, *args = line.split()
        if kind == "thread":
            events = roles[args[0]] = []
        elif kind == "name":
            names[int(args[0])] = args[1]
        elif kind == "init":
            counts[int(args[0])] = int(args[1])
        else:
            events.append((kind, *(int(a) if a.lstrip("-").isdigit() else a for a in args)))
    for role, events in roles.items():
        syncs = [i for i, e in enumerate(events) if e[0] == "sync"]
        assert len(syncs) == 2, role
        roles[role] = events[syncs[0] + 1:syncs[1]]
    assert set(names) == set(counts)
    # of the threads that arrive on a barrier, those that are traced
    traced = {1: 1, 128: warps, 4: warps, 3 + 8: 4 - 1 + 2 * warps}
    return roles, names, {b: traced[n] for b, n in counts.items()}


def _programs(roles, names, D, warps):
    """Each role's steps: ("wait", bar, parity), ("arrive", bar), ("touch", accesses), and ("start", pipe, operations): copies and MMAs
    under way from here on.  An access is (place, whether it writes); an operation (accesses, barrier or None, arrivals, copies)."""
    tile = 128 * D * 2
    everyone = range(warps)

    def smem(address):                                  # of a query tile, or a slot of the ring
        i = address // tile
        return [("Q", i, w) for w in everyone] if i < 2 else [("KV", i - 2)]

    def of(accesses, writes=False):
        return [(place, writes) for place in accesses]

    described = {name: sorted(b for b in names if names[b] == name) for name in ("seg_full", "seg_empty")}
    programs = {}
    for role, events in roles.items():
        program, i = [], 0
        few = False                                     # the tile in hand is one of few rows
        while i < len(events):
            kind, *a = events[i]
            i += 1
            if kind == "wait":
                program.append(("wait", *a))
            elif kind == "arrive":
                if few and names[a[0]] == "p_lo":       # P of few rows lies in the second query tile
                    program.append(("touch", [(("Q", 1, int(role[-1])), True)]))
                    few = False
                if names[a[0]] in described:            # a description of a unit, written and read
                    program.append(("touch", [(("unit", described[names[a[0]]].index(a[0])), names[a[0]] == "seg_full")]))
                program.append(("arrive", a[0]))
            elif kind == "expect":                      # with the copies behind it
                places = []
                while i < len(events) and events[i][0] == "load" and events[i][3] == a[0]:
                    places += [p for p in smem(events[i][1]) if p not in places]
                    i += 1
                assert places, role
                program.append(("start", "copies", [(of(places, True), a[0], 0, 1)]))
            elif kind in ("qk", "pv"):
                d, x, y, _ = a
                reads = smem(y) + (smem(x) if kind == "qk" else [("P", (x - 128) // 32, w) for w in everyone])
                place = [("S",)] if d < 128 else [("O", d // 128 - 2, w) for w in everyone]
                op = (of(reads) + of(place, True), None, 0, 0)
                if program and program[-1][0] == "start" and program[-1][2][-1] == op:
                    continue                            # the same tiles, further along
                program.append(("start", role, [op]))
            elif kind == "commit":
                program.append(("start", role, [([], a[0], 1, 0)]))
            elif kind == "stage":
                program.append(("touch", of(smem(a[0]), True)))
            elif kind in ("ld", "st"):
                col, width = a
                t, w = int(role[5]), int(role[-1])
                few |= kind == "ld" and width == 16 and col < 128
                place = ("S",) if col < 128 else ("P", (col - 128) // 32, w) if col < 256 else ("O", t, w)
                if col >= 256:
                    assert col // 128 - 2 == t
                program.append(("touch", [(place, kind == "st")]))
            else:
                assert kind in ("before", "after", "wait_st", "dealloc"), kind
        programs[role] = program
    return programs


# ------------------------------------------------------------------------------------------------------------------ execution
class Block:
    def __init__(self, programs, names, counts):
        self.programs, self.names, self.counts = programs, names, counts
        self.follows = None

    def run(self, choose):
        """Runs to the end; ``choose`` picks one of the actors that can take a step."""
        at = dict.fromkeys(self.programs, 0)
        bars = {b: [0, n, 0] for b, n in self.counts.items()}      # phase, arrivals and copies that it waits for
        queues = {"copies": [], "scores": [], "values": []}
        last, follows = {}, {}

        def settle(bar):
            if bars[bar][1] < 0:
                raise Wrong(f"{self.names[bar]}: an arrival too many")
            if bars[bar][1] == 0 and bars[bar][2] == 0:
                bars[bar] = [bars[bar][0] + 1, self.counts[bar], 0]

        def touch(accesses, key):
            for n, (place, writes) in enumerate(accesses):
                before = follows[key, n] = last.get(place)
                if self.follows is not None and self.follows.get((key, n)) != before:
                    raise Wrong(f"{place} touched at the wrong time by {key[0]}")
                if writes:
                    last[place] = (key, n)

        while True:
            ready = []
            for role, program in self.programs.items():
                if at[role] < len(program):
                    step = program[at[role]]
                    if step[0] != "wait" or (bars[step[1]][0] & 1) != step[2]:
                        ready.append(role)
            ready += [">" + q for q, ops in queues.items() if ops]
            if not ready:
                break
            actor = choose(ready)
            if actor[0] == ">":
                ops = queues[actor[1:]]
                key, (accesses, bar, arrivals, copies) = ops.pop(0 if actor != ">copies" else choose.which(len(ops)))
                touch(accesses, key)
                if bar is not None:
                    bars[bar][1] -= arrivals
                    bars[bar][2] -= copies
                    settle(bar)
                continue
            step, key = self.programs[actor][at[actor]], (actor, at[actor])
            at[actor] += 1
            if step[0] == "arrive":
                bars[step[1]][1] -= 1
                settle(step[1])
            elif step[0] == "touch":
                touch(step[1], key)
            elif step[0] == "start":
                for n, op in enumerate(step[2]):
                    queues[step[1]].append(((">" + actor, key[1], n), op))
                    if op[3]:                           # the copy's bytes are announced with an arrival
                        bars[op[1]][1] -= 1
                        bars[op[1]][2] += 1
                        settle(op[1])
        stuck = sorted({self.names[p[at[r]][1]] for r, p in self.programs.items() if at[r] < len(p)})
        if stuck:
            raise Wrong(f"stuck, waiting for {stuck}")
        if self.follows is None:
            self.follows = follows


class InOrder:
    """The first of a list of actors that can take a step."""

    def __init__(self, order, newest=False):
        self.rank = {a: i for i, a in enumerate(order)}
        self.newest = newest

    def __call__(self, ready):
        return min(ready, key=self.rank.__getitem__)

    def which(self, n):
        return n - 1 if self.newest else 0


class AtRandom:
    """Any actor, a few steps at a time, some of them slower than others."""

    def __init__(self, rng, actors):
        self.rng, self.speed = rng, {a: rng.choice([1, 1, 5, 60]) for a in actors}

    def __call__(self, ready):
        return self.rng.choices(ready, [self.speed[a] for a in ready])[0]

    def which(self, n):
        return self.rng.randrange(n)


def _run(program, units, *, D=128, kernel="thin", mode="steady", G=4, warps=1, orders=40):
    """What goes wrong with these units in some order, or None."""
    roles, names, counts = _trace(program, D, kernel, mode, G, warps, units)
    block = Block(_programs(roles, names, D, warps), names, counts)
    actors = [*block.programs, ">copies", ">scores", ">values"]
    rng = random.Random(len(units))
    try:
        block.run(InOrder([">copies", ">scores", ">values", *reversed(block.programs)]))
        for actor, last in itertools.product(actors, (True, False)):          # each as late, and as early, as it can be
            others = [a for a in actors if a != actor]
            for order in (others, others[::-1], rng.sample(others, len(others))):
                block.run(InOrder(order + [actor] if last else [actor] + order, newest=rng.random() < 0.5))
        for _ in range(orders):
            block.run(InOrder(rng.sample(actors, len(actors)), newest=rng.random() < 0.5))
            block.run(AtRandom(rng, actors))
    except Wrong as e:
        return str(e)
    return None


# ------------------------------------------------------------------------------------------------------------------------ tests
# new tokens and length of each sequence, a unit each: at G = 4 up to 4 tokens are few rows, 32 a query tile, 64 two
FEW, FEW_LONG, TILE, TWO, TWO_LONG, EMPTY, NONE = (1, 100), (4, 300), (30, 200), (64, 120), (50, 400), (1, 0), (0, 77)


@pytest.mark.parametrize("empty", [0, 1, 2, 14, 15, 16, 17, 33])
def test_units_without_keys_between_few_rows_and_a_chunk(built, empty):
    assert _run(built(), [FEW, FEW] + [EMPTY] * empty + [TWO, FEW]) is None


@pytest.mark.parametrize("units", [
    [FEW], [TWO], [EMPTY], [TILE, TILE], [TWO, TWO, FEW], [FEW, TWO, FEW, TWO, TWO], [FEW, TILE, TWO], [FEW_LONG, TILE, TILE, TWO_LONG],
    [FEW, FEW_LONG, FEW, TWO, TWO_LONG, FEW, EMPTY, TWO], [TWO, EMPTY, FEW, EMPTY, TWO], [FEW] * 18 + [TWO], [FEW] + [EMPTY] * 17 + [TILE, TWO],
    [TWO] + [EMPTY] * 17 + [TWO], [FEW, NONE, NONE, TWO], [TILE] * 17 + [FEW, TWO] + [EMPTY] * 20 + [FEW, TWO_LONG],
], ids=lambda u: "-".join(f"{n}of{kv}" for n, kv in u[:4]) + f"-{len(u)}")
@pytest.mark.parametrize("kernel", ["thin", "thick"])
def test_units_of_all_kinds(built, units, kernel):
    assert _run(built(), units, kernel=kernel) is None


@pytest.mark.parametrize("kernel", ["thin", "thick"])
@pytest.mark.parametrize("D, mode, warps", [(64, "steady", 1), (128, "growing", 2), (64, "growing", 2)])
def test_forms(built, kernel, D, mode, warps):
    """Heads of 64 channels (ten slots of the ring), offsets that move at every tile, two warps of a group out of step."""
    assert _run(built(), [FEW_LONG, TWO_LONG, FEW, EMPTY, FEW, TILE, TWO], D=D, kernel=kernel, mode=mode, warps=warps) is None


def test_batches_drawn_at_random(built):
    rng = random.Random(7)
    for _ in range(12):
        units = [rng.choice([FEW, FEW, FEW_LONG, TILE, TWO, TWO_LONG, EMPTY, EMPTY, NONE]) for _ in range(rng.randint(2, 40))]
        assert _run(built(), units, orders=15) is None, units


MISTAKES = {
    # the producer and the memory that few-row units share with the second query tile
    "one barrier for all units, two phases of it waited for in turn": [
        ("return &bars->o_free[t][n & 1];", "return &bars->o_free[t][0];"), ("{ return (n >> 1) & 1; }", "{ return n & 1; }"),
        ("ok = warp_wait(o_free_of(bars, 0, n_q - 1), o_free_parity(n_q - 1), ctx, SITE_PG_QE);",
         "if (n_q > 1) ok = warp_wait(&bars->o_free[0][0], n_q & 1, ctx, SITE_PG_QE);\n if (ok) ok = warp_wait(&bars->o_free[0][0], (n_q - 1) & 1, ctx, SITE_PG_QE);")],
    "one barrier for all units, one phase of it": [("return &bars->o_free[t][n & 1];", "return &bars->o_free[t][0];"), ("{ return (n >> 1) & 1; }", "{ return n & 1; }")],
    "the second query tile copied over P": [("ok = warp_wait(o_free_of(bars, 0, n_q - 1), o_free_parity(n_q - 1), ctx, SITE_PG_QE);", "")],
    "a unit of few rows forgotten": [("thin_before |= kThin && s.ntok * p.G <= kThinRows;", "thin_before = kThin && s.ntok * p.G <= kThinRows && s.ntok > 1;")],
    # between units
    "Q copied before it is read": [("if (n_q > 0) ok = warp_wait(&bars->q_empty, (n_q - 1) & 1, ctx, SITE_PG_QE);", "")],
    "Q not waited for": [("ok = warp_wait(&bars->q_full, n_q & 1, ctx, SITE_PG_Q);", "")],
    "units without keys counted as over": [("n_o += s.n_tiles > 0;", "++n_o;")],
    "a description overwritten while a warp has not read it": [("ok = mbar_wait(smem_u32(&bars->seg_empty[w.i % kSegs]), (w.i / kSegs - 1) & 1, ctx, SITE_PG_SEGE);", "ok = true;")],
    # within a unit
    "S overwritten before it is read": [("if (n_s > 0) ok = warp_wait(&bars->s_free, (n_s - 1) & 1, ctx, SITE_PG_SF);", "")],
    "a slot reloaded before it is free": [("if (use > 0) ok = warp_wait(&bars->kv_empty[slot], (use - 1) & 1, ctx, SITE_PG_KVE);", "")],
    "P written before the last product": [("const bool done = warp_wait(&bars->pv_done[t], (count - 2) & 1, ctx, SITE_PG_O);", "const bool done = true;")],
    "P of few rows written before the last product": [("const bool done = warp_wait(&bars->pv_done[0], (count - 2) & 1, ctx, SITE_PG_O);", "const bool done = true;")],
    "O of few rows read before the last product": [("if (!warp_wait(&bars->pv_done[0], (count - 1) & 1, ctx, SITE_PG_O)) return -1;", "")],
}


@pytest.mark.parametrize("mistake", MISTAKES)
def test_a_planted_mistake_is_found(built, mistake):
    program = built(tuple(MISTAKES[mistake]))
    batches = [FEW, FEW, TWO, FEW, TWO], [FEW] + [EMPTY] * 18 + [TWO, TWO], [FEW_LONG, TWO_LONG, FEW, EMPTY, FEW, TILE, TWO], [FEW, FEW_LONG, FEW, FEW] + [TILE] * 20
    assert any(_run(program, units, warps=warps, mode="growing") for warps in (1, 2) for units in batches)
