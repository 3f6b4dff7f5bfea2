"""CPU: the scan's check of shared memory against the sets of addresses themselves."""
import random

import torch

from vdn_b200.recurrence import _beside, _meets


def _addresses(t):
    at = torch.zeros(t.shape, dtype=torch.long) + t.storage_offset()
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([n if i == d else 1 for i in range(t.dim())])
    return set(at.flatten().tolist())


def test_views_that_pass_share_no_address():
    rng, buffer, apart, refused = random.Random(0), torch.zeros(5000), 0, 0
    for _ in range(4000):
        lead = rng.choice([1, 2])
        shape = [rng.choice([1, 2, 3, 4]) for _ in range(lead)]
        steps = [[rng.choice([1, 2, 4, 6, 8, 12, 16, 24, 48, 96]) for _ in range(lead)] for _ in range(2)]
        if rng.random() < 0.8:
            steps[1] = steps[0]
        a, b = (buffer.as_strided(shape + [width], step + [1], rng.randrange(far))
                for width, step, far in zip((rng.choice([1, 2, 4, 6]), rng.choice([1, 2, 4, 6])), steps, (40, 200)))
        if not _meets(a, b) or _beside(a, b, lead):
            assert not _addresses(a) & _addresses(b)
            apart += 1
        else:
            refused += not _addresses(a) & _addresses(b)
    assert apart > 3000 and refused < 300                  # odd lattices that it cannot tell apart are refused
