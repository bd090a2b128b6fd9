"""Workspaces of the losses on logits, without a GPU."""


def test_the_policy_workspace_of_many_short_rows_follows_their_blocks():
    """Four sums in 64 bits a block of at least four rows, not a position: 1 GB and not 4 at the most positions."""
    from mote_b200 import _lib as L
    size = lambda n, V: L.lib.moteopt_policy_loss_workspace_size(L.Logits(256, 1, 1, n, V, 0, V))  # noqa: E731
    for n in (50_000, 15_900_000, 2 ** 27 - 1):
        assert 8 * n <= size(n, 271) <= 8 * n + 8192
        assert 32 * n <= size(n, 5000) <= 32 * n + 8192   # a block or more a row
    for n in (1, 3, 1000, 4096):
        assert size(n, 271) >= 32 * n
