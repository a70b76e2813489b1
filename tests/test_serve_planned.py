"""The loop of the serving example over tables on the device, with a layer that computes nothing (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")


class Layer:
    """Steps of a layer whose free pages end at some step: rows of zeros and a status word, as the GPU's."""

    def __init__(self, fails):
        self.torch, self.n_seqs, self.status, self.fails = torch, 3, torch.zeros(1, dtype=torch.int32), fails
        self.steps, self.ended = 0, []

    def step_planned(self, x, rows):
        assert len(x) == sum(rows)
        if self.steps == self.fails:
            self.status |= 32
        self.steps += 1
        return torch.zeros_like(x)

    def normed(self, y):
        return y

    def end(self, sequences):
        self.ended += list(sequences)


def test_a_step_without_room_is_an_error(l2):
    import paged_serving
    prompts = [torch.ones(n, 8) for n in (3, 30, 9)]
    layer = Layer(-1)
    outs, steps, rows = paged_serving.serve_planned(layer, prompts, 2, 8)
    assert [len(o) for o in outs] == [5, 32, 11] and rows == 48 and sorted(layer.ended) == [0, 1, 2]
    for fails in range(steps):
        layer = Layer(fails)
        with pytest.raises(RuntimeError, match="status 32"):
            paged_serving.serve_planned(layer, prompts, 2, 8)
        assert set(layer.ended) == {0, 1, 2}  # the pages come back
