"""A map that places points no fit has seen.

t-SNE moves the points it is given; it has no place for a later one.
``ParametricMap`` learns one: an encoder whose distribution over the fitted
points (``softmax`` of the logarithms of Student's kernel between where it puts
a point and where they are) is distilled from the point's own neighbour
probabilities.  The encoder's wide layers run on 8-bit products of bfloat16
activations and float32 weights (``operators.block_linear`` in training, with
float32 gradients of the weights, ``operators.linear_blocks`` on weights quantised
once afterwards), the neighbours' probabilities are the teacher's list of
``operators.distill_loss``.

    embedding = TSNE(...).fit_transform(X)
    mapping = ParametricMap().fit(X, embedding)
    placed = mapping.transform(X_later)
"""
import math

import numpy as np
import torch

from . import operators, stages

_MOST_DISTANCES = 1 << 25


class ParametricMap(object):
    """Encoder from input space into a finished embedding.

    hidden         widths of the encoder's layers (8-bit products, ReLU)
    num_neighbors, perplexity, perplexity_epsilon   as in ``TSNE``: the teacher's lists
    batch_size, n_epochs, learning_rate             of the training (Adam)
    random_seed    of the initial weights and the order of the points
    """

    def __init__(self, hidden=(1024, 1024), num_neighbors=32, perplexity=10.0, perplexity_epsilon=1e-3, batch_size=512,
                 n_epochs=40, learning_rate=1e-3, random_seed=0, gpu_device=0):
        if len(hidden) < 1 or any(int(h) < 1 for h in hidden):
            raise ValueError("hidden must be the widths of one layer or more (got %r)" % (hidden,))
        if batch_size < 1 or n_epochs < 0 or not learning_rate > 0:
            raise ValueError("batch_size and learning_rate must be positive and n_epochs not negative")
        if not 2 <= num_neighbors <= operators.MAX_LISTED:
            raise ValueError("num_neighbors must be in [2, %d] (got %d)" % (operators.MAX_LISTED, num_neighbors))
        self.hidden = tuple(int(h) for h in hidden)
        self.num_neighbors, self.perplexity = num_neighbors, perplexity
        self.perplexity_epsilon = perplexity_epsilon
        self.batch_size, self.n_epochs, self.learning_rate = batch_size, n_epochs, learning_rate
        self.random_seed = random_seed
        self.device = torch.device("cuda", gpu_device)
        self.losses_ = None

    def _points(self, X):
        X = torch.as_tensor(np.ascontiguousarray(X, dtype=np.float32) if not isinstance(X, torch.Tensor) else X)
        if X.dim() != 2:
            raise ValueError("points must be a matrix (got shape %s)" % (tuple(X.shape),))
        return X.detach().to(self.device, torch.float32).contiguous()

    def _scaled(self, X):
        return ((X - self._mean) * self._scale).to(torch.bfloat16)

    def _hidden(self, x):
        for w in self._weights:
            x = torch.relu(operators.block_linear(x, w))
        return x

    def _head(self, h):
        return h.to(torch.float32) @ self._last.t() + self._bias

    def _logits(self, y):
        """Logarithms of Student's kernel between the places y and the fitted points'."""
        square = (y[:, :1] - self._anchors[:, 0]) ** 2 + (y[:, 1:] - self._anchors[:, 1]) ** 2
        return -torch.log1p(square)

    def fit(self, X, embedding):
        """Trains the encoder on points X (n x d) and the embedding (n x 2) that a fit gave them; n at most 2^20.
        Afterwards ``losses_`` holds the mean divergence of every epoch."""
        X = self._points(X)
        embedding = self._points(embedding)
        n, d = X.shape
        if tuple(embedding.shape) != (n, 2):
            raise ValueError("the embedding of %d points must be of shape (%d, 2) (got %s)" % (n, n, tuple(embedding.shape)))
        if not self.num_neighbors <= n <= operators.MAX_DISTILLED:
            raise ValueError("fit takes num_neighbors (%d) to %d points (got %d)" % (self.num_neighbors, operators.MAX_DISTILLED, n))
        self.losses_ = None  # (until there is a map again)
        with torch.cuda.device(self.device), torch.enable_grad():
            # The teacher: what the fit's own stages say of the points.  (A point's own entry has probability 0.)
            indices, square = stages.knn(X, self.num_neighbors)
            pij = stages.perplexity(stages.max_normalize_(square), self.perplexity, self.perplexity_epsilon)
            values = torch.log(pij)
            self._anchors = embedding.clone()
            self._mean = X.mean(0)
            self._scale = 1.0 / (X - self._mean).std().clamp(min=1e-30)
            x = self._scaled(X)
            g = torch.Generator(device=self.device)
            g.manual_seed(self.random_seed)
            widths = (d,) + self.hidden
            self._weights = [(torch.randn(o, i, generator=g, device=self.device) * math.sqrt(2.0 / i)).requires_grad_()
                             for i, o in zip(widths[:-1], widths[1:])]
            spread = embedding.std(0)
            self._last = (torch.randn(2, widths[-1], generator=g, device=self.device) / math.sqrt(widths[-1])
                          * spread[:, None]).requires_grad_()
            self._bias = embedding.mean(0).clone().requires_grad_()
            optimiser = torch.optim.Adam(self._weights + [self._last, self._bias], lr=self.learning_rate)
            losses = []
            batches = -(-n // self.batch_size)
            for epoch in range(self.n_epochs):
                order = torch.randperm(n, generator=g, device=self.device)
                for group in optimiser.param_groups:
                    group["lr"] = self.learning_rate * 0.5 * (1 + math.cos(math.pi * epoch / self.n_epochs))
                total = torch.zeros((), device=self.device)
                for b in range(batches):
                    rows = order[b * self.batch_size:(b + 1) * self.batch_size]
                    y = self._head(self._hidden(x[rows]))
                    # The rest of the embedding is far from a new point's first places, and its pull weak there: the mean
                    # distance to where the fit put the point leads, while there are epochs left to lead for.
                    lead = max(0.0, 1.0 - 2.0 * epoch / self.n_epochs)
                    loss = operators.distill_loss(self._logits(y), indices[rows], values[rows]).mean()
                    if lead:
                        near = (((y - embedding[rows]) / spread.mean()) ** 2).sum(1).mean()
                        (loss + 10.0 * lead * near).backward()
                    else:
                        loss.backward()
                    optimiser.step()
                    optimiser.zero_grad(set_to_none=True)
                    total += loss.detach() * rows.numel()
                losses.append(total / n)
            self._quantized = [operators.quantize_blocks(w.detach(), square=True) for w in self._weights]
            self.losses_ = [float(v) for v in losses]
        return self

    def _check_fitted(self):
        if self.losses_ is None:
            raise ValueError("fit() comes before places can be asked for")

    def _place(self, X):
        X = self._points(X)
        if X.shape[1] != self._mean.numel():
            raise ValueError("points of %d dimensions (the fit's had %d)" % (X.shape[1], self._mean.numel()))
        h = self._scaled(X)
        for w in self._quantized:
            h = torch.relu(operators.linear_blocks(h, w))
        return self._head(h)

    def transform(self, X):
        """Places (m x 2, float32) of points X (m x d), one or many: a numpy array, or a tensor for a tensor."""
        self._check_fitted()
        with torch.cuda.device(self.device), torch.no_grad():
            y = self._place(X)
        return y if isinstance(X, torch.Tensor) else y.cpu().numpy()

    def neighbors(self, X, k=10):
        """(probabilities, indices), m x k each: the fitted points that X's points lie nearest to in the map, and the
        shares of the map's own distribution that they hold."""
        self._check_fitted()
        with torch.cuda.device(self.device), torch.no_grad():
            y = self._place(X)
            # So many rows at a time that their distances to all fitted points are 128 MB.
            rows = max(1, _MOST_DISTANCES // len(self._anchors))
            tops = [operators.top_logits(self._logits(y[r:r + rows]), k) for r in range(0, max(1, len(y)), rows)]
            p = torch.cat([torch.exp(top.values - top.lse[:, None]) for top in tops])
            i = torch.cat([top.indices for top in tops])
        return (p, i) if isinstance(X, torch.Tensor) else (p.cpu().numpy(), i.cpu().numpy())
