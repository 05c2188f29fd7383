"""Model of the warps that store a product's tiles and of the bounded waits ahead of each (csrc/kernels/gemm_int8.cu ``i8_epilogue``, gemm_rows.cuh
``rows_epilogue``).

For every tile a warp waits until the tile's sums are complete, at most for a time of its own, then stores the tile together with the other warps of its
group, between barriers of that group; after its last tile it meets all warps of the block.  The wait of one warp may run out just before the sums are
there while another's still sees them.  What has to hold: whatever the waits do, every warp reaches the end of the kernel.

``vote=False`` lets each warp go by its own wait: the search finds a warp that skips the tile and others that stay in the group's barrier.
``owes=True`` lets it, too, but sends the warp through all barriers that it has not been in yet (csrc/kernels/attention_fp8_tc.cu, one a block of keys and
one behind them), which costs nothing where no wait runs out.
"""
from __future__ import annotations

from ..utils.model_check import Result, explore


def check(warps: int = 4, tiles: int = 2, barriers: int = 2, vote: bool = True, owes: bool = False) -> Result:
    # A warp: (tile, place, ok, went).  place 0: waits; 1: meets the group for the vote; 2 .. barriers + 1: the group's barriers; "end": the block's.
    # complete: how many tiles' sums are there.
    init = (((0, 0, True, False),) * warps, 0)

    def after(tile, ok):
        return (tile + 1, 0, ok, False) if tile + 1 < tiles else (tiles, "end", ok, False)

    def step(s):
        state, complete = s
        if complete < tiles:
            yield ("sums", (state, complete + 1))
        for i, (tile, place, ok, _) in enumerate(state):
            if place != 0:
                continue
            ends = []
            if ok and complete > tile:
                ends.append(("sees", True))
            if not ok or complete <= tile:
                ends.append(("gives up", False))
            for what, seen in ends:
                # one that gave up before waits no longer and, with a vote, does not ask for another
                if owes:
                    nxt = (tile, 2, ok and seen, seen)
                elif not ok or not (vote or seen):
                    nxt = after(tile, False)
                elif vote:
                    nxt = (tile, 1, ok, seen)
                else:
                    nxt = (tile, 2, ok, seen)
                yield (f"warp{i} {what} {tile}", (state[:i] + (nxt,) + state[i + 1:], complete))
        # a barrier lets its warps go when all of them are in it, wherever in the program they stand
        if all(w[1] not in (0, "end") for w in state):
            went = all(w[3] for w in state)
            nxt = []
            for tile, place, ok, seen in state:
                if place == 1:
                    nxt.append((tile, 2, ok, seen) if went else after(tile, False))
                else:
                    nxt.append((tile, place + 1, ok, seen) if place <= barriers else after(tile, ok))
            yield ("barrier", (tuple(nxt), complete))

    return explore(init, step, {"the group is at one tile": lambda s: len({(w[0], w[1]) for w in s[0] if w[1] not in (0, "end")}) <= 1},
                   lambda s: all(w[1] == "end" for w in s[0]))
