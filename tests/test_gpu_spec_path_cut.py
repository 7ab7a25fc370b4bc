"""Paths that path_stride cuts off: the last row's children have no part in the draw, whether
they would have stood or not."""
import numpy as np
import pytest
import torch

from test_gpu_spec_verify import Verify
from tree_cases import lines, verify_oracle

pytestmark = pytest.mark.gpu


class Cut(Verify):
    """Against the definition over the rows that a path can reach at all: those at a depth of path_stride and more
    hang on none, so that no path has to be cut off."""

    def check(self):
        keep = self.chain, self.parent
        self.chain, self.parent = False, self.reached()
        try:
            return super().check()
        finally:
            self.chain, self.parent = keep

    def reached(self):
        parent = self.parent.copy()
        for r0, n in zip(self.start[:-1].astype(int), self.n):
            for i, line in enumerate(lines(self.parent[r0:r0 + n])):
                if len(line) > self.path:
                    parent[r0 + i] = -1
        return parent

    def rejected(self):
        """Requests whose path is cut off where none of the children would have stood: by the same inputs with longer paths."""
        x = self.target[:, :self.vocab].double().numpy()
        y = self.draft[:, :self.vocab].double().numpy() if self.draft is not None else None
        n_path = verify_oracle(x, y, self.start, self.token, self.parent, self.inv_temp, self.u_accept, self.u_next, max(self.n),
                               self.max_child, self.vocab)[0]
        ends = n_path == self.path
        for s in np.nonzero(ends)[0]:
            r0 = int(self.start[s])
            deep = [len(line) for line in lines(self.parent[r0:r0 + self.n[s]])]
            ends[s] = max(deep) > self.path
        return int(ends.sum())


def case(flh, s, path, kids, draft, seed):
    v = Cut(flh, s, [9, 13, 2, 21, 1, 30, 0] + [9, 40, 17] * 9, 700, "F32", draft, kids, seed=seed, path=path, peak=3.0)
    v.u_accept[np.random.default_rng(seed).random(v.rows) < 0.6] = 1e-6  # (these stand if they are likely at all)
    return v


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("kids", [1, 3])
@pytest.mark.parametrize("path", [1, 2, 3])
def test_cut_off(flh, gpu, path, kids, draft):
    bites = 0
    for seed in range(3):
        v = case(flh, gpu, path, kids, draft, seed)
        v.push().run()
        v.check()
        bites += v.rejected()
    assert bites >= 2


@pytest.mark.parametrize("path", [1, 2, 7])
@pytest.mark.parametrize("draft", [False, True])
def test_distributed_as_the_target(flh, gpu, draft, path):
    """The first token that comes out, and the second one where a drafted token stood in front of it, are distributed
    as p, wherever the path is cut off: 6 standard deviations of a count."""
    n, vocab = 30000, 6
    rng = np.random.default_rng(41)
    v = Verify(flh, gpu, [7] * n, vocab, "F32", draft, 2, seed=41, chain=False, temp=False, path=path)
    x, y = np.array([0.0, 1.0, -1.0, 0.5, -3.0, 0.2]), np.array([1.5, -1.0, 0.3, 0.0, 1.0, -0.5])
    v.target[:, :vocab] = torch.from_numpy(x).float()
    p, q = np.exp(x) / np.exp(x).sum(), np.exp(y) / np.exp(y).sum()
    if draft:
        v.draft[:, :vocab] = torch.from_numpy(y).float()
    v.token[:] = rng.choice(vocab, v.rows, p=q)
    v.push().run()
    n_path, path_, nxt, _, _ = v.read()
    assert n_path.max() == min(path, 3)
    tokens = np.full((n, 4), -1, np.int64)
    for j in range(1, min(path, 3)):
        on = n_path > j
        tokens[on, j - 1] = v.token[v.start[:-1][on] + path_[on, j]]
    tokens[np.arange(n), n_path.astype(int) - 1] = nxt
    for j in range(min(path, 2)):
        seen = tokens[:, j][tokens[:, j] >= 0]
        m, counts = len(seen), np.bincount(seen, minlength=vocab)
        assert m > 5000 and (np.abs(counts - m * p) <= 6 * np.sqrt(m * p * (1 - p))).all(), (j, counts, m * p)
