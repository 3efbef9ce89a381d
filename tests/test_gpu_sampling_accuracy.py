"""GPU: `sample` over the longest rows by uniform numbers next to the borders between tokens, and min-p among very small weights.

A running sum of n logits is off by their roundings to units of 2^-f and 2^-38 of itself (derived in test_sampling_weights.py): by n / 2 units at
most, and as independent roundings, a twelfth of a unit squared each, within eight standard deviations by 8 sqrt(n / 12)."""
import numpy as np
import pytest
import torch

from triton_amd.sampling import sample

pytestmark = pytest.mark.gpu
V, F = 1 << 20, 41


@pytest.mark.parametrize("rows", [1, 24])
def test_tokens_next_to_a_border(rows, device):
    """Of a million uniform numbers those that lie nearest to a border between two tokens, but twice as far as the sums may be off."""
    z = 2.5 * torch.randn(V, generator=torch.Generator().manual_seed(11))
    order = np.argsort(-z.double().numpy(), kind="stable")
    c = np.cumsum(np.exp(z.double().numpy()[order].astype(np.longdouble) - z.max().item()))
    u = np.random.default_rng(3).integers(1, 1 << 24, 1 << 20).astype(np.float64) / (1 << 24)
    at = u * c[-1]
    token = np.searchsorted(c, at, side="right")
    low = np.where(token > 0, c[token - 1], -1.0)
    distance = np.minimum(c[token] - at, at - low)
    # the border's running sum and u times the sum of all are off by as much each
    least = 2 * (8 * np.sqrt(V / 12) * 2.0**-F + 2.0**-38 * c[-1])
    usable = np.flatnonzero(distance > least)
    nearest = usable[np.argsort(distance[usable])[:240]]
    assert distance[nearest].max() < 2.0**-29 * c[-1]   # (as near as the sums would be off if weights were cut off instead of rounded)
    want = order[token[nearest]].tolist()
    numbers = torch.from_numpy(u[nearest]).float().to(device)
    logits = z.to(device).expand(rows, V)
    got = torch.cat([sample(logits[:n.shape[0]], n) for n in numbers.split(rows)]).tolist()
    assert got == want


def test_a_tail_of_weights_below_two_units(device):
    """One logit holds nearly all, the others weigh 1.97 units each: the token is the definition's up to what n / 2 units amount to."""
    weight = 1.97
    z = torch.full((3, V), float(np.log(weight * 2.0**-F)), device=device)
    z[:, 0] = 0.0
    w = np.exp(z[0, 1].double().item()) * 2.0**F
    u = torch.tensor([1.0 - 2.0**-24, 1.0 - 4 * 2.0**-24, 1.0 - 7 * 2.0**-24], device=device)
    got = sample(z, u).cpu().double().numpy()          # (equal logits: a token's place in the order is its index)
    total = 2.0**F + (V - 1) * w
    reached, asked = 2.0**F + got * w, u.cpu().double().numpy() * total
    assert (got > 0).all() and (np.abs(reached - asked) <= V / 2 + w + 2.0**-38 * total).all()


@pytest.mark.parametrize("rows", [40, 300])
@pytest.mark.parametrize("tail", [60000, V - 1])
def test_min_p_among_very_small_weights(tail, rows, device):
    """What has w >= min_p is kept, also where weights are a few units, whether the row is searched or sorted, alone or shared out.  Weights spread
    evenly over whole units round to either side alike; of a range that begins or ends inside a unit the part of that unit does not, and of tail / 12 weights
    to a unit half a unit's lose or gain at most an eighth of a unit each: tail / 96 at either end."""
    g = np.random.default_rng(tail)
    z = torch.full((V,), -float("inf"))
    z[torch.from_numpy(g.permutation(V)[:tail + 1])] = torch.from_numpy(np.log(np.concatenate([[2.0**F], g.uniform(2.5, 14.5, tail)]) * 2.0**-F)).float()
    order = np.argsort(-z.double().numpy(), kind="stable")
    w = np.exp(z.double().numpy()[order].astype(np.longdouble)) * 2.0**F
    min_p = torch.from_numpy(np.linspace(3.1, 13.9, rows) * 2.0**-F).float()
    u = 1.0 - 2.0**-24
    got = sample(z.to(device).expand(rows, V), torch.full((rows,), u, device=device), min_p=min_p.to(device)).tolist()
    place = np.empty(V, np.int64)
    place[order] = np.arange(V)
    for t, m in zip(got, min_p.double().numpy() * 2.0**F):
        c = np.cumsum(w[:int((w >= m).sum())])
        off = 2 * (8 * np.sqrt(len(c) / 12) + tail / 96 + 2.0**-38 * c[-1])   # of the token's running sum and of the sum of all
        at = place[t]
        assert at < len(c) and c[at] + off >= u * c[-1] and (c[at - 1] if at else 0.0) - off <= u * c[-1]
