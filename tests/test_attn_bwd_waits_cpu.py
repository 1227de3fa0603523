"""The waits of the attention's backward kernels (csrc/attn_bwd.cu, csrc/attn_bwd_gather.cu), modelled on the CPU.

Every warp, or group of warps with one role, is a list of steps: wait for a phase of a barrier, arrive at one, write a place, read a place
and find what was meant for it.  Barriers behave as the hardware's: a wait sees the parity of the running phase only, so a barrier that has
moved two phases on looks as if it had not moved.  A run holds one warp up in front of one of its steps until nobody else can go on, then
lets it go; every step of every warp is held up once.  No run may get stuck or read what was not meant for the reader.

The models follow the kernels' program order by hand.  Each switch takes one of the kernel's waits away, and the model has to find
what that wait is for.
"""

import pytest


class Barrier:
    def __init__(self, count):
        self.count, self.pending, self.phases = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.phases = self.count, self.phases + 1


class Fault(Exception):
    pass


class Model:
    def __init__(self):
        self.counts, self.warps = {}, {}

    def barrier(self, name, count):
        self.counts[name] = count

    def warp(self, name):
        steps = self.warps[name] = []
        return (lambda bar, phase: steps.append(("wait", bar, phase)), lambda bar: steps.append(("arrive", bar, None)),
                lambda place, value: steps.append(("write", place, value)), lambda place, value: steps.append(("read", place, value)))

    def run(self, held, at):
        bars = {name: Barrier(n) for name, n in self.counts.items()}
        places, pos = {}, dict.fromkeys(self.warps, 0)

        def advance(name, stop):
            """Steps of a warp until it has to wait; whether it took any."""
            steps, first = self.warps[name], pos[name]
            while pos[name] < stop:
                op, what, value = steps[pos[name]]
                if op == "wait" and bars[what].phases & 1 == value & 1:
                    break
                if op == "arrive":
                    bars[what].arrive()
                elif op == "write":
                    places[what] = value
                elif op == "read" and places.get(what) != value:
                    raise Fault(f"{name} reads {what}: {places.get(what)} for {value} (held: {held} at {at})")
                pos[name] += 1
            return pos[name] > first

        for stops in ({held: at}, {}):
            while any([advance(name, stops.get(name, len(steps))) for name, steps in self.warps.items()]):
                pass
        stuck = {n: steps[pos[n]] for n, steps in self.warps.items() if pos[n] < len(steps)}
        if stuck:
            raise Fault(f"stuck (held: {held} at {at}): {stuck}")

    def check(self):
        for name, steps in self.warps.items():
            for at in range(len(steps)):
                self.run(name, at)


def backward(items, keys, ordered, ring, gather=False, ordered_sums=True, all_arrive=True):
    """One CTA of attn_bwd_kernel that walks `items` (tiles of each).  `keys`: the mode of dK and dV, else that of dQ.  `ordered`: tiles of 128
    rows, whose S and dP are issued in a fixed order.  `gather`: six warps copy batches of 32 rows in turn, instead of two that issue TMA.
    The eight softmax warps are two: the halves of the columns."""
    m = Model()
    batches = (4 if ordered else 2) if gather else 1
    res_batches = 8 if gather else 1
    for name, count in dict(a_full=res_batches, a_empty=2, s_full=1, s_free=2, dp_full=1, p_ready=2, ds_ready=2, o_full=1, o_free=2, row_sum=2).items():
        m.barrier(name, count)
    for i in range(ring):
        m.barrier(("full", i), batches + (GATHER_WARPS if gather and all_arrive else 0))
        m.barrier(("empty", i), 1)
    tiles = [(ic, t, t == n - 1) for ic, n in enumerate(items) for t in range(n)]

    def full(wait, load):
        wait(("full", load % ring), load // ring)

    def read_tile(read, load):
        for q in range(batches):
            read(("ring", load % ring, q), load)

    def read_resident(read, ic):
        for q in range(res_batches):
            read(("A", q), ic)

    for x in range(2):
        wait, arrive, write, read = m.warp(f"softmax {x}")
        for g, (ic, t, last) in enumerate(tiles):
            n0, n1 = 2 * g, 2 * g + 1
            wait("s_full", g)
            if keys:
                full(wait, n0)
            read("S", g)
            arrive("s_free")
            if keys:
                read(("statistics", n0 % ring), n0)
            wait("dp_full", g)
            if keys:
                full(wait, n1)
            read("dP", g)
            write(("P", x), g)
            arrive("p_ready")
            if keys:
                read(("statistics", n1 % ring), n1)
            write(("dS", x), g)
            arrive("ds_ready")
            if not last:
                continue
            if not keys:
                if ordered_sums and ic > 0:
                    wait("o_free", ic - 1)
                write(("sums", x), ic)
                arrive("row_sum")
                wait("row_sum", ic)
                read(("sums", 1 - x), ic)
            wait("o_full", ic)
            read("sum of P", ic)
            read("sum of dS", ic)
            arrive("o_free")

    wait, arrive, write, read = m.warp("scores")
    for g, (ic, t, last) in enumerate(tiles):
        if t == 0:
            wait("a_full", ic)
        full(wait, 2 * g)
        if ordered and t > 0:
            wait("dp_full", g - 1)
        if g > 0:
            wait("s_free", g - 1)
        read_resident(read, ic)
        read_tile(read, 2 * g)
        write("S", g)
        arrive("s_full")
        if last:
            arrive("a_empty")

    wait, arrive, write, read = m.warp("sums")
    for g, (ic, t, last) in enumerate(tiles):
        n0, n1 = 2 * g, 2 * g + 1
        if t == 0:
            wait("a_full", ic)
        if ordered and t > 0:
            wait("s_full", g)
        full(wait, n1)
        read_resident(read, ic)
        read_tile(read, n1)
        write("dP", g)
        arrive("dp_full")
        if not keys:
            arrive(("empty", n1 % ring))
        if last:
            arrive("a_empty")
        wait("p_ready", g)
        if t == 0 and ic > 0:
            wait("o_free", ic - 1)
        n = n1 if keys else n0
        read_tile(read, n)
        for x in range(2):
            read(("P", x), g)
        write("sum of P", ic)
        if keys:
            # (the deltas of this slot may still be wanted; the ring is loaded in order, and T0's slot comes first)
            arrive(("empty", n1 % ring))
        wait("ds_ready", g)
        for x in range(2):
            read(("dS", x), g)
        read_tile(read, n0)
        write("sum of dS", ic)
        arrive(("empty", n0 % ring))
        if last:
            arrive("o_full")

    if gather:
        for w in range(GATHER_WARPS):
            wait, arrive, write, read = m.warp(f"rows {w}")
            n = batch = 0
            for ic, t, last in tiles:
                for n in (n, n + 1):
                    if n >= ring:
                        wait(("empty", n % ring), n // ring - 1)
                    for q in range(batches):
                        if batch % GATHER_WARPS == w:
                            write(("ring", n % ring, q), n)
                            arrive(("full", n % ring))
                        batch += 1
                    if all_arrive:
                        arrive(("full", n % ring))
                n += 1
                if t == 0:
                    if ic > 0:
                        wait("a_empty", ic - 1)
                    for q in range(res_batches):
                        if batch % GATHER_WARPS == w:
                            write(("A", q), ic)
                            arrive("a_full")
                        batch += 1
        return m
    wait, arrive, write, read = m.warp("resident tiles")
    for ic in range(len(items)):
        if ic > 0:
            wait("a_empty", ic - 1)
        write(("A", 0), ic)
        arrive("a_full")
    wait, arrive, write, read = m.warp("ring")
    for n in range(2 * len(tiles)):
        if n >= ring:
            wait(("empty", n % ring), n // ring - 1)
        write(("ring", n % ring, 0), n)
        write(("statistics", n % ring), n)
        arrive(("full", n % ring))
    return m


GATHER_WARPS = 6
ITEMS = [(1, 1, 1, 1), (1, 2, 1, 3, 1), (3, 1, 1, 2), (5, 4)]
# (rows of a tile are 128 with rings of 5 and 8 tiles, or 64 with 5 and 3)
SHAPES = [(True, 5), (True, 8), (False, 5), (False, 3)]


@pytest.mark.parametrize("ordered,ring", SHAPES)
@pytest.mark.parametrize("items", ITEMS)
@pytest.mark.parametrize("keys", [False, True])
def test_dense_modes(items, keys, ordered, ring):
    backward(items, keys, ordered, ring).check()


@pytest.mark.parametrize("ordered,ring", SHAPES)
def test_row_sums_of_an_item_of_one_tile_wait_for_the_reads_of_the_item_before(ordered, ring):
    with pytest.raises(Fault, match="sums"):
        backward((1, 1, 1, 1), False, ordered, ring, ordered_sums=False).check()
    backward((2, 2, 2), False, ordered, ring, ordered_sums=False).check()       # (the sum of the first tile's P orders the second's dP)


@pytest.mark.parametrize("ordered,ring", SHAPES)
@pytest.mark.parametrize("items", [*ITEMS, (4, 1, 1, 5), (7, 1, 3)])
def test_gathered_keys(items, ordered, ring):
    backward(items, False, ordered, ring, gather=True).check()


@pytest.mark.parametrize("ordered,ring", SHAPES)
def test_a_warp_without_rows_of_a_load_has_a_part_in_it_all_the_same(ordered, ring):
    """Without its arrival the load is consumed, and the slot's barrier moves on, before the warp has seen the phase that it waits for."""
    with pytest.raises(Fault, match="stuck"):
        for items in ((4, 1, 1, 5), (7, 1, 3), (1, 1, 1, 1, 1, 1, 1)):
            backward(items, False, ordered, ring, gather=True, all_arrive=False).check()


def contributions(items, blocks, ring):
    """One CTA of attn_bwd_gather_dkv_kernel that walks groups of `items` tiles, `blocks` column blocks of 128: softmax warps by halves of the
    columns, the issuer, three warps that copy rows, the warps that copy out as one."""
    m = Model()
    for name, count in dict(a_full=8, a_empty=1, s_full=1, dp_full=1, p_ready=2, ds_ready=2, dv_full=1, dv_free=1, dk_full=1, dk_free=1).items():
        m.barrier(name, count)
    for i in range(ring):
        m.barrier(("full", i), 4)
        m.barrier(("empty", i), 1)
    tiles = [(ic, t, t == n - 1) for ic, n in enumerate(items) for t in range(n)]

    for x in range(2):
        wait, arrive, write, read = m.warp(f"softmax {x}")
        for g, (ic, t, last) in enumerate(tiles):
            if t == 0:
                wait("a_full", ic)
            wait("s_full", g)
            read(("S", x), g)
            read(("A", 0), ic)                               # statistics come with the first rows
            write(("S", x), ("P", g))
            arrive("p_ready")
            wait("dp_full", g)
            read(("dP", x), g)
            read(("A", 4), ic)
            write(("dP", x), ("dS", g))
            arrive("ds_ready")

    wait, arrive, write, read = m.warp("issuer")
    n = block = 0
    for g, (ic, t, last) in enumerate(tiles):
        if t == 0:
            wait("a_full", ic)
        for name, done in (("S", "s_full"), ("dP", "dp_full")):
            for cb in range(blocks):
                wait(("full", n % ring), n // ring)
                for q in range(4):
                    read(("ring", n % ring, q), n)
                for q in range(8):
                    read(("A", q), ic)
                for x in range(2):
                    write((name, x), g)
                arrive(("empty", n % ring))
                n += 1
            arrive(done)
        wait("p_ready", g)
        for cb in range(blocks):
            if block > 0:
                wait("dv_free", block - 1)
            for x in range(2):
                read(("S", x), ("P", g))
            for q in range(8):
                read(("A", q), ic)
            write("dV", block)
            arrive("dv_full")
            if cb == 0:
                wait("ds_ready", g)
            if block > 0:
                wait("dk_free", block - 1)
            for x in range(2):
                read(("dP", x), ("dS", g))
            write("dK", block)
            arrive("dk_full")
            block += 1
        if last:
            arrive("a_empty")

    for w in range(3):
        wait, arrive, write, read = m.warp(f"rows {w}")
        n = batch = 0
        for ic, t, last in tiles:
            for e in range(2 * blocks):
                if n >= ring:
                    wait(("empty", n % ring), n // ring - 1)
                for q in range(4):
                    if batch % 3 == w:
                        write(("ring", n % ring, q), n)
                        arrive(("full", n % ring))
                    batch += 1
                if t == 0 and e == 0:
                    if ic > 0:
                        wait("a_empty", ic - 1)
                    for q in range(8):
                        if batch % 3 == w:
                            write(("A", q), ic)
                            arrive("a_full")
                        batch += 1
                n += 1

    wait, arrive, write, read = m.warp("copy out")
    for block in range(len(tiles) * blocks):
        for name, full, free in (("dV", "dv_full", "dv_free"), ("dK", "dk_full", "dk_free")):
            wait(full, block)
            read(name, block)
            arrive(free)
    return m


@pytest.mark.parametrize("blocks,ring", [(1, 8), (1, 4), (2, 2)])
@pytest.mark.parametrize("items", [*ITEMS, (4, 1, 1, 5)])
def test_contributions_of_gathered_keys(items, blocks, ring):
    contributions(items, blocks, ring).check()
