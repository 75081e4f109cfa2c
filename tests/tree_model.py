"""Trees of drafted tokens for the tests: random trees and what follows from their parents, on the host."""
import numpy as np

NO = 0xffffffff


def random_tree(rng, n, width=4, chain=0.0):
    """Parents of n nodes: node 0 the root, none with more than `width` children."""
    parent, count = [-1][:n], [0]
    for i in range(1, n):
        p = i - 1 if rng.random() < chain else int(rng.integers(0, i))
        while count[p] >= width:
            p = (p + 1) % i
        parent.append(p)
        count.append(0)
        count[p] += 1
    return parent


def lines(parent):
    """Per node the list of its ancestors and itself, from the root down. A parent that is not in front is none."""
    out = []
    for i, p in enumerate(parent):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def masks(parent):
    return np.array([sum(1 << j for j in line) for line in lines(parent)], np.uint64)


def starts(nodes):
    return np.concatenate([[0], np.cumsum(nodes)]).astype(np.int64)


def flat(forest, pad=0):
    return np.array([p & NO for parent in forest for p in parent] + [NO] * pad, np.uint32)
