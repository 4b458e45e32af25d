"""Pages and slots of a batch by a loop over its sequences, as whole numbers."""


def reserve(table, lens, new, free, count, page, total, finished=None):
    """``table`` rows and ``free`` are changed; (q_starts, kv_lens, free_count, positions, slots)."""
    width, cap = len(table[0]) if table else 0, (len(table[0]) if table else 0) * page
    up = lambda x: -(-x // page)
    clamp = lambda x, hi: min(max(x, 0), hi)
    count = clamp(count, len(free))
    old = [clamp(l, cap) for l in lens]
    new = [clamp(n, total) for n in new]
    if finished is not None:
        for s, ended in enumerate(finished):
            if not ended:
                continue
            for c in range(min(up(old[s]), width)):
                if table[s][c] >= 0 and count < len(free):
                    free[count] = table[s][c]
                    count += 1
            old[s] = 0
    starts, positions, slots, wanted = [0], [-1] * total, [-1] * total, 0
    for s, n in enumerate(new):
        for c in range(min(up(old[s]), width), min(up(old[s] + n), width) if n else 0):
            at = count - 1 - wanted
            table[s][c] = free[at] if at >= 0 else -1
            wanted += 1
        for i in range(n):
            t, place = starts[-1] + i, old[s] + i
            if t >= total:
                break
            pg = table[s][place // page] if place // page < width else -1
            positions[t] = place
            slots[t] = -1 if pg < 0 else pg * page + place % page
        starts.append(starts[-1] + n)
    return starts, [o + n for o, n in zip(old, new)], max(count - wanted, 0), positions, slots
