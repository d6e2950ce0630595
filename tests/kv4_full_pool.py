"""Growth of the 4-bit cache's sequences where the pool runs out, one entry after the other, and what has to hold after it."""
import numpy as np


def resize_in_order(a, page, seq, new_len):
    """Statuses and copies (source, destination, rows) of mk_kv4_resize; a: table, len, refs, changed in place. An entry copies its
    last page where somebody holds that page beside it when its turn comes. What it wants is kept for it, or missing, also where
    it does not get it."""
    n_seq, max_pages = a["table"].shape
    seq = list(range(len(new_len))) if seq is None else [int(s) for s in seq]
    good = [0 <= s < n_seq and 0 <= L <= max_pages * page and s not in seq[i + 1:] for i, (s, L) in enumerate(zip(seq, new_len))]
    had = {s: int(a["len"][s]) for s, ok in zip(seq, good) if ok}
    for s, L, ok in zip(seq, new_len, good):
        if ok and L <= had[s]:
            first = -(-L // page)
            for p in a["table"][s, first:-(-had[s] // page)]:
                a["refs"][p] -= 1
            a["table"][s, first:] = -1
            a["len"][s] = L
    free = list(np.flatnonzero(a["refs"] <= 0))
    status, copies, used = [0 if ok else -1 for ok in good], [], 0
    for i, (s, L) in enumerate(zip(seq, new_len)):
        if not good[i] or L <= had[s]:
            continue
        at, part = divmod(had[s], page)
        p = int(a["table"][s, at]) if part else -1
        copy = part > 0 and a["refs"][p] > 1
        places = ([at] if copy else []) + list(range(-(-had[s] // page), -(-L // page)))
        first, used = used, used + len(places)
        if places and used > len(free):
            status[i] = 1
            continue
        if copy:
            copies.append((p, int(free[first]), part))
            a["refs"][p] -= 1
        a["table"][s, places] = free[first:used]
        a["refs"][free[first:used]] += 1
        a["len"][s] = L
    return status, copies


def written_pages(a, page, seq, before, status):
    """(sequence, page) of every page that an entry of status 0 may write rows to now."""
    for s, st in zip(range(len(status)) if seq is None else seq, status):
        if st == 0:
            for j in range(int(before[s]) // page, -(-int(a["len"][s]) // page)):
                yield s, int(a["table"][s, j])
