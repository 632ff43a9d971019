"""The batched 64-bit form against the one that takes one sequence after the other."""
import pytest
import torch

import seq_batched
import seq_reference as ref


@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('bare', [False, True])
def test_batched_scan_is_the_single_one(reverse, bare):
    T, n, Dn, G, N = 6, 5, 4, 2, 3
    g = torch.Generator().manual_seed(1)
    f = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)             # noqa: E731
    acts = dict(u=f(T, n, Dn), delta=f(T, n, Dn), B=f(T, n, G, N), Cm=f(T, n, G, N), z=None if bare else f(T, n, Dn), gy=f(T, n, Dn))
    par = dict(A=-f(Dn, N).abs(), D=None if bare else f(Dn), bias=None if bare else f(Dn))
    init = None if bare else f(n, Dn, N)
    want = ref.by_sequence(ref.scan_one, acts, dict(init=init), [T] * n, False, reverse, ('y', 'gu', 'gdelta', 'gz', 'gB', 'gC'), ('gA', 'gD', 'gbias'), par)
    for got in (seq_batched.scan(**acts, **par, init=init, reverse=reverse), seq_batched.scan_in_chunks(2, **acts, **par, init=init, reverse=reverse)):
        assert set(got) == set(want)
        for k in want:
            for a, b in zip(got[k], want[k]):
                torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-13)
