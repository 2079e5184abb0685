"""The map for later points: what it refuses, and where it puts points that the fit has not seen."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tsnecuda.parametric import ParametricMap  # noqa: E402


def test_refusals():
    for how in (dict(hidden=()), dict(hidden=(0,)), dict(batch_size=0), dict(learning_rate=0.0), dict(num_neighbors=1),
                dict(num_neighbors=1025), dict(n_epochs=-1)):
        with pytest.raises(ValueError):
            ParametricMap(**how)
    with pytest.raises(ValueError, match="fit"):
        ParametricMap().transform(np.zeros((3, 4), np.float32))


@pytest.fixture(scope="module")
def fitted():
    from tsnecuda import TSNE, synthetic
    X = synthetic.gaussian_clusters(4000, d=50, clusters=8, center_scale=3.0, seed=5)
    seen = X[:3000]
    embedding = TSNE(perplexity=20.0, num_neighbors=48, n_iter=500).fit_transform(
        seen, y=synthetic.initial_embedding(3000, seed=6))
    mapping = ParametricMap(hidden=(256, 200), num_neighbors=48, perplexity=20.0, n_epochs=20)
    return X, embedding, mapping.fit(seen, embedding)


@pytest.mark.gpu
def test_later_points_lie_with_their_own(fitted):
    X, embedding, mapping = fitted
    assert len(mapping.losses_) == 20 and np.isfinite(mapping.losses_).all()
    # Training closes half of what lies between its first epoch and the divergence of the places that the fit gave.
    from tsnecuda import operators, stages
    seen = torch.from_numpy(X[:3000]).cuda()
    indices, square = stages.knn(seen, 48)
    values = torch.log(stages.perplexity(stages.max_normalize_(square), 20.0, 1e-3))
    own = torch.from_numpy(np.ascontiguousarray(embedding)).cuda()
    least = float(operators.distill_loss(mapping._logits(own), indices, values).mean())
    assert mapping.losses_[-1] - least < 0.5 * (mapping.losses_[0] - least), (mapping.losses_, least)
    placed = mapping.transform(X[3000:])
    assert placed.shape == (1000, 2) and placed.dtype == np.float32
    labels = np.arange(4000) % 8  # (as synthetic.gaussian_clusters numbers them)
    p, idx = mapping.neighbors(X[3000:], k=10)
    assert (labels[idx] == labels[3000:, None]).mean() > 0.95
    # The list is the nearest of the map, and its shares are the kernel's.
    square = ((placed[:, None].astype(np.float64) - embedding[None]) ** 2).sum(2)
    kernel = 1 / (1 + square)
    share = kernel / kernel.sum(1, keepdims=True)
    np.testing.assert_allclose(p, np.take_along_axis(share, idx, 1), rtol=1e-3)
    np.testing.assert_allclose(p, -np.sort(-share, 1)[:, :10], rtol=1e-3)


@pytest.mark.gpu
def test_one_point_is_placed_as_among_many(fitted):
    X, _, mapping = fitted
    many = mapping.transform(X[3000:])
    for i in (0, 17, 999):
        one = mapping.transform(X[3000 + i:3001 + i])
        # (other kernels, other orders of 32-bit sums: what that does to a hidden value is a rounding of bfloat16, 2^-8)
        assert np.abs(one[0] - many[i]).max() <= 2.0 ** -6 * np.abs(many).max()
    as_tensor = mapping.transform(torch.from_numpy(X[3000:]).cuda())
    assert as_tensor.is_cuda and np.array_equal(as_tensor.cpu().numpy(), many)


@pytest.mark.gpu
def test_the_same_seed_trains_the_same_map(fitted):
    X, embedding, _ = fitted
    how = dict(hidden=(130,), num_neighbors=20, perplexity=5.0, n_epochs=2)
    maps = [ParametricMap(**how).fit(X[:600], embedding[:600]) for _ in range(2)]
    assert np.allclose(maps[0].losses_, maps[1].losses_, rtol=1e-4)
    with pytest.raises(ValueError, match="dimensions"):
        maps[0].transform(X[:, :40])
    with pytest.raises(ValueError, match="shape"):
        maps[0].fit(X[:600], embedding[:500])
    with pytest.raises(ValueError, match="num_neighbors"):
        maps[0].fit(X[:10], embedding[:10])


@pytest.mark.gpu
def test_weights_are_rounded_once(monkeypatch):
    """The encoder's float32 weights become 8-bit ones directly, in training and afterwards, and their gradients are float32."""
    from tsnecuda import operators, synthetic
    X = synthetic.gaussian_clusters(600, d=50, clusters=8, center_scale=3.0, seed=7)
    embedding = synthetic.initial_embedding(600, seed=8)
    seen, block_linear = [], operators.block_linear
    monkeypatch.setattr(operators, "block_linear", lambda x, w: seen.append(w.dtype) or block_linear(x, w))
    mapping = ParametricMap(hidden=(200, 130), num_neighbors=20, perplexity=5.0, n_epochs=2).fit(X, embedding)
    assert set(seen) == {torch.float32}
    for w, q in zip(mapping._weights, mapping._quantized):
        want = operators.quantize_blocks(w.detach(), square=True)
        assert torch.equal(q.data.view(torch.uint8), want.data.view(torch.uint8))
        assert torch.equal(q.scales.view(torch.uint8), want.scales.view(torch.uint8))


@pytest.mark.gpu
def test_a_fit_that_fails_leaves_no_map(fitted, monkeypatch):
    from tsnecuda import operators
    X, embedding, _ = fitted
    mapping = ParametricMap(hidden=(130,), num_neighbors=20, perplexity=5.0, n_epochs=1).fit(X[:600], embedding[:600])
    with pytest.raises(ValueError, match="shape"):  # (refused before anything is done: the map stays)
        mapping.fit(X[:600], embedding[:500])
    assert mapping.transform(X[:3]).shape == (3, 2)

    def fails(*args, **how):
        raise RuntimeError("no memory")

    monkeypatch.setattr(operators, "distill_loss", fails)
    for which in (mapping, ParametricMap(hidden=(130,), num_neighbors=20, perplexity=5.0, n_epochs=1)):
        with pytest.raises(RuntimeError, match="no memory"):
            which.fit(X[:600], embedding[:600])
        assert which.losses_ is None
        for ask in (which.transform, which.neighbors):
            with pytest.raises(ValueError, match="fit"):
                ask(X[:3])


@pytest.mark.gpu
def test_neighbors_of_many_points_take_little_memory(fitted):
    X, _, mapping = fitted
    many = torch.from_numpy(np.tile(X, (30, 1))).cuda()  # 120,000 points by 3000 places: 1.4 GB of distances
    mapping.neighbors(many[:100], k=5)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    p, i = mapping.neighbors(many, k=5)
    taken = torch.cuda.max_memory_allocated() - before
    assert p.shape == i.shape == (120000, 5)
    # (the points and hidden values as bfloat16 and floats are 120,000 x 256 x a few bytes)
    assert taken < 1 << 30, taken
    for a in (0, 4000, 116000):
        q, j = mapping.neighbors(many[a:a + 4000], k=5)
        assert torch.allclose(p[a:a + 4000], q, rtol=0.05) and (i[a:a + 4000] == j).float().mean() > 0.95
    empty = mapping.neighbors(many[:0], k=5)
    assert empty[0].shape == empty[1].shape == (0, 5)


@pytest.mark.gpu
def test_a_map_is_its_own(fitted):
    """What a caller does with the embedding afterwards, or wants gradients of, or has switched off, is nothing to the map."""
    X, embedding, _ = fitted
    how = dict(hidden=(130,), num_neighbors=20, perplexity=5.0, n_epochs=1)
    places = torch.from_numpy(np.ascontiguousarray(embedding[:600])).cuda()
    mapping = ParametricMap(**how).fit(X[:600], places)
    p, i = mapping.neighbors(X[600:700], k=5)
    places.zero_()
    q, j = mapping.neighbors(X[600:700], k=5)
    assert np.array_equal(p, q) and np.array_equal(i, j)
    with torch.no_grad():
        again = ParametricMap(**how).fit(X[:600], embedding[:600])
    assert np.allclose(again.losses_, mapping.losses_, rtol=1e-4)
    points = torch.from_numpy(X[:600].copy()).cuda().requires_grad_()
    again = ParametricMap(**how).fit(points, embedding[:600])
    assert points.grad is None and np.allclose(again.losses_, mapping.losses_, rtol=1e-4)
    assert not again.transform(points).requires_grad
