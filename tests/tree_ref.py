"""Trees of drafted tokens in 64 bits."""
import torch

TREES = {
    "one": [-1],
    "chain5": [-1, 0, 1, 2, 3],
    "star7": [-1] * 7,
    "binary15": [-1] + [(j - 1) // 2 for j in range(1, 15)],
    "two_roots": [-1, -1, 0, 1, 2, 3, 0, 1, 6],
    "chain64": list(range(-1, 63)),
    "wide63": [-1, 0, 0, 0] + [1 + j % 3 for j in range(59)],
}


def random_tree(n, seed):
    tree, x = [], seed * 7919 + 17
    for j in range(n):
        x = (x * 1103515245 + 12345) % (1 << 31)
        tree.append((x >> 12) % (j + 1) - 1)
    return tree


def tree_of(spec):
    return TREES[spec] if isinstance(spec, str) else random_tree(*spec) if isinstance(spec, tuple) else list(spec)


def path(tree, j):
    """a node's ancestors from the root on, itself last; a parent that is no earlier node is none"""
    out = []
    while j >= 0:
        out.insert(0, j)
        p = tree[j]
        j = p if 0 <= p < j else -1
    return out


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def layout(trees, front=0):
    """(first rows, parent, tree_start): `front` rows of no tree first"""
    starts = [front]
    for t in trees:
        starts.append(starts[-1] + len(t))
    return starts, ints([0] * front + [p for t in trees for p in t] or [0]), ints(starts)


def kda_token(s, q, k, v, g, b):
    """one token on the states [heads][128][128] in 64 bits: (state, output)"""
    q, k = (x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    s = s * torch.exp(g)[..., None]
    u = (v - torch.einsum("hk,hkv->hv", k, s)) * b[:, None]
    s = s + torch.einsum("hk,hv->hkv", k, u)
    return s, torch.einsum("hk,hkv->hv", q, s) * 128 ** -0.5
