"""scikit-learn style estimators: the public API of the framework.

Mirrors the reference's estimator surface (``mpitree/tree/decision_tree.py``):
``DecisionTreeClassifier(*, max_depth=None, min_samples_split=2)`` with
``fit``/``predict_proba``/``predict``/``export_text`` (:17-307) and the
collective ``ParallelDecisionTreeClassifier`` (:310-479), plus the
regression tree and extra hyperparameters the BASELINE configurations need
(``criterion``, ``max_bins``, ``min_samples_leaf``, ``device``, ``strategy``).

Behavioural contract kept from the reference:

* ``predict_proba`` returns the leaf's raw per-class **counts** (int64), not
  normalised probabilities (reference :192-227); pass ``normalize=True`` for
  probabilities.
* ``predict`` is the argmax of those counts with ties to the lowest class,
  returned as the class label (the reference returns the class index, which
  is the same whenever labels are ``0..K-1``).
* ``tree_`` is the linked ``Node`` graph; pickles carry the reference state
  keys and module paths, so checkpoints load in either framework.

Internally a fitted estimator holds flat arrays (:class:`TreeArrays`);
``tree_`` is materialised lazily.
"""

from __future__ import annotations

import os

import numpy as np
import torch
from sklearn.base import BaseEstimator, ClassifierMixin, RegressorMixin
from sklearn.utils.validation import check_is_fitted

from ..core.criterion import parse_criterion
from ..core.fit import fit_tree
from ..ops.leaf_ops import LeafRoute, leaf_embedding, leaf_linear, leaf_route
from .tree_arrays import TreeArrays
from ..utils.level_checkpoint import CheckpointInterrupt

# errors a rank raises from its own state, never from a collective a failed peer
# broke: a rank keeps them even when a peer's failure reached it first (ranks
# that fail alike -- invalid input, a checkpoint stop -- each report their own)
_OWN_ERRORS = (ValueError, TypeError, CheckpointInterrupt)

__all__ = [
    "DecisionTreeClassifier",
    "DecisionTreeRegressor",
    "ParallelDecisionTreeClassifier",
    "ParallelDecisionTreeRegressor",
]

_STATE_SKIP = ("_arrays", "_tree_cache", "_device_tree", "fit_result_")


def _as_numpy_X(X):
    if isinstance(X, torch.Tensor):
        return X.detach().cpu().numpy()
    X = np.asarray(X)
    if X.dtype == object:
        X = X.astype(np.float64)
    return X


class _BaseTree(BaseEstimator):
    _regression = False

    def __init__(
        self,
        *,
        max_depth: int | None = None,
        min_samples_split: int = 2,
        criterion: str = "entropy",
        min_samples_leaf: int = 1,
        max_bins: int | None = None,
        device: str = "auto",
    ):
        self.max_depth = max_depth
        self.min_samples_split = min_samples_split
        self.criterion = criterion
        self.min_samples_leaf = min_samples_leaf
        self.max_bins = max_bins
        self.device = device

    # ------------------------------------------------------------------ fit
    def _fit_impl(self, X, y, comm=None, **kw):
        crit = parse_criterion(self.criterion, regression=self._regression)
        res = fit_tree(
            X,
            y,
            regression=self._regression,
            criterion=crit,
            max_depth=self.max_depth,
            min_samples_split=self.min_samples_split,
            min_samples_leaf=self.min_samples_leaf,
            max_bins=self.max_bins,
            device=self.device,
            comm=comm,
            **kw,
        )
        self._arrays = res.arrays
        self.n_features_ = int(res.n_features)
        self.n_features_in_ = int(res.n_features)
        if not self._regression:
            self.classes_ = res.classes
        self.fit_stats_ = {
            "engine": res.engine,
            "timings": res.timings,
            **res.stats,
            "node_count": res.arrays.node_count,
            "max_depth": res.arrays.max_depth,
            "n_leaves": res.arrays.n_leaves,
        }
        self._tree_cache = None
        self._device_tree = None
        return self

    def fit(self, X, y, *, checkpoint=None):
        """Grow the tree on ``X`` (n, F) and targets ``y`` (n,).

        ``checkpoint``: a file path; the grower (the GPU's device level loop or
        the level-wise builder) saves its state there after every level and a
        re-run of the same fit resumes from the last saved level
        (``utils/level_checkpoint.py``)."""
        if checkpoint is not None:
            return self._fit_impl(X, y, checkpoint=checkpoint)
        return self._fit_impl(X, y)

    # ------------------------------------------------------------ tree views
    @property
    def tree_arrays_(self) -> TreeArrays:
        check_is_fitted(self, "n_features_")
        return self._arrays

    @property
    def tree_(self):
        check_is_fitted(self, "n_features_")
        if getattr(self, "_tree_cache", None) is None:
            self._tree_cache = self._arrays.to_nodes(
                getattr(self, "classes_", None), regression=self._regression
            )
        return self._tree_cache

    def get_depth(self) -> int:
        return self.tree_arrays_.max_depth

    def get_n_leaves(self) -> int:
        return self.tree_arrays_.n_leaves

    # ------------------------------------------------------------ inference
    def _check_X_predict(self, X):
        if isinstance(X, torch.Tensor):
            if X.dim() != 2:
                raise ValueError("Expected 2D input")
            nf = X.shape[1]
        else:
            X = _as_numpy_X(X)
            if X.ndim != 2:
                raise ValueError(f"Expected 2D array, got {X.ndim}D array instead")
            nf = X.shape[1]
        if nf != self.n_features_:
            raise ValueError(
                f"X has {nf} features, but {type(self).__name__} is expecting "
                f"{self.n_features_} features as input"
            )
        return X

    def apply(self, X):
        """Index (pre-order) of the leaf each row reaches."""
        check_is_fitted(self, "n_features_")
        X = self._check_X_predict(X)
        if isinstance(X, torch.Tensor) and X.is_cuda:
            from ..ops.hip_predict import predict_leaves

            return predict_leaves(self, X)
        return self._arrays.apply(_as_numpy_X(X))

    # ----------------------------------------------- learned leaf parameters
    def _leaf_numbers(self, X):
        check_is_fitted(self, "n_features_")
        X = self._check_X_predict(X)
        if isinstance(X, torch.Tensor) and X.is_cuda:
            from ..ops.hip_predict import leaf_numbers

            return leaf_numbers(self, X)
        return torch.from_numpy(self._arrays.leaf_numbers()[self._arrays.apply(_as_numpy_X(X))])

    def _leaves_for(self, X, what, params):
        """Leaf numbers (or the route) of ``X`` on the parameters' device."""
        check_is_fitted(self, "n_features_")
        if not isinstance(params, torch.Tensor) or params.dim() < 1:
            raise TypeError(f"{what} must be a tensor with one entry per leaf")
        if params.shape[0] != self.get_n_leaves():
            raise ValueError(f"{what} has {params.shape[0]} entries, the tree "
                             f"{self.get_n_leaves()} leaves")
        if isinstance(X, LeafRoute):
            return X
        return self._leaf_numbers(X).to(params.device)

    def leaf_route(self, X) -> LeafRoute:
        """The rows of ``X`` sorted by the leaf they reach. The leaf operators below take it in
        place of ``X``: a fitted tree's rows do not change leaves, so a training loop over the
        leaves' parameters walks and sorts them once."""
        return leaf_route(self._leaf_numbers(X), self.get_n_leaves())

    def leaf_embedding(self, X, table, *, scale: float = 1.0):
        """``scale * table[leaf]`` for the leaf of each row: ``table`` is a float tensor
        [n_leaves, D], leaves numbered in pre-order; differentiable in ``table``
        (:func:`mpitree_amd.leaf_embedding`). ``X``: rows, or their :meth:`leaf_route`."""
        return leaf_embedding(self._leaves_for(X, "table", table), table, scale=scale)

    def leaf_linear(self, X, weight, bias=None, *, inputs=None):
        """A linear model per leaf: ``inputs[i] @ weight[leaf].T + bias[leaf]``, with ``weight``
        [n_leaves, N, K] and ``bias`` [n_leaves, N]; differentiable in all three
        (:func:`mpitree_amd.leaf_linear`). ``inputs`` (n, K) defaults to the rows ``X`` themselves,
        in the weight's type. ``X``: rows, or their :meth:`leaf_route` (then give ``inputs``)."""
        leaves = self._leaves_for(X, "weight", weight)
        if inputs is None:
            if isinstance(X, LeafRoute):
                raise ValueError("a LeafRoute holds no features: pass inputs")
            rows = X
            if not isinstance(X, torch.Tensor):  # (torch takes no reversed or foreign-endian ones)
                rows = _as_numpy_X(X)
                rows = torch.from_numpy(np.require(rows, rows.dtype.newbyteorder("="), "CW"))
            inputs = rows.to(device=weight.device, dtype=weight.dtype)
        return leaf_linear(inputs, leaves, weight, bias)

    # --------------------------------------------------------------- export
    def export_text(self, *, feature_names=None, class_names=None, precision=2) -> str:
        """Text rendering identical to the reference's ``export_text``."""
        check_is_fitted(self, "n_features_")
        return self._arrays.export_text(
            feature_names=feature_names,
            class_names=class_names,
            precision=precision,
            classes=getattr(self, "classes_", None),
            regression=self._regression,
        )

    # ---------------------------------------------------------- persistence
    def __getstate__(self):
        state = {k: v for k, v in self.__dict__.items() if k not in _STATE_SKIP}
        if "_arrays" in self.__dict__:
            state["tree_"] = self.tree_
        return state

    def __setstate__(self, state):
        state = dict(state)
        state.pop("_sklearn_version", None)
        tree = state.pop("tree_", None)
        self.__dict__.update(state)
        # parameters added by this framework default when loading reference pickles
        defaults = {"criterion": "squared_error" if self._regression else "entropy",
                    "min_samples_leaf": 1, "max_bins": None, "device": "auto"}
        for k, v in defaults.items():
            self.__dict__.setdefault(k, v)
        if tree is not None:
            self._arrays = TreeArrays.from_nodes(
                tree, getattr(self, "classes_", None), regression=self._regression
            )
            self._tree_cache = tree
        self._device_tree = None

    def save(self, path):
        """Pickle the estimator (the reference's checkpoint format)."""
        from ..utils.checkpoint import save

        save(self, path)

    @classmethod
    def load(cls, path):
        from ..utils.checkpoint import load

        return load(path)


class DecisionTreeClassifier(_BaseTree, ClassifierMixin):
    """Decision tree classifier (entropy or gini), exact thresholds.

    Parameters
    ----------
    max_depth : int, optional
        Maximum depth (``None`` grows until leaves are pure).
    min_samples_split : int, default=2
        Nodes with fewer rows become leaves.
    criterion : {"entropy", "gini"}, default="entropy"
    min_samples_leaf : int, default=1
    max_bins : int or None, default=None
        ``None`` (default): every unique value of a feature is a candidate
        threshold, exactly the reference's search (``decision_tree.py:73``).
        An int opts into quantile binning: features with at most this many
        unique values stay exact, others get ``max_bins`` quantile edges
        (every edge a data value).
    device : {"auto", "cpu", "cuda"}, default="auto"
    """

    _regression = False

    def predict_proba(self, X, normalize: bool = False):
        """Leaf class counts (reference semantics) or probabilities.

        Device-tensor inputs are answered on the device (torch tensors out).
        """
        leaves = self.apply(X)
        if isinstance(leaves, torch.Tensor):
            counts = torch.from_numpy(self._arrays.count).to(leaves.device)[leaves].long()
            if normalize:
                return counts.double() / counts.sum(1, keepdim=True)
            return counts
        counts = self._arrays.count[leaves].astype(np.int64, copy=False)
        if normalize:
            return counts / counts.sum(axis=1, keepdims=True)
        return counts

    def predict(self, X):
        leaves = self.apply(X)
        lab = self._arrays.leaf_label_index()
        if isinstance(leaves, torch.Tensor):
            if np.issubdtype(np.asarray(self.classes_).dtype, np.number):
                table = torch.from_numpy(np.asarray(self.classes_)[lab]).to(leaves.device)
                return table[leaves]
            leaves = leaves.cpu().numpy()
        return self.classes_[lab[leaves]]


class DecisionTreeRegressor(_BaseTree, RegressorMixin):
    """Regression tree with the squared-error (MSE) criterion."""

    _regression = True

    def __init__(
        self,
        *,
        max_depth: int | None = None,
        min_samples_split: int = 2,
        criterion: str = "squared_error",
        min_samples_leaf: int = 1,
        max_bins: int | None = None,
        device: str = "auto",
    ):
        super().__init__(
            max_depth=max_depth,
            min_samples_split=min_samples_split,
            criterion=criterion,
            min_samples_leaf=min_samples_leaf,
            max_bins=max_bins,
            device=device,
        )

    def predict(self, X):
        leaves = self.apply(X)
        if isinstance(leaves, torch.Tensor):
            return torch.from_numpy(self._arrays.value).to(leaves.device)[leaves]
        return self._arrays.value[leaves]


class _WorldAttr:
    """Class-and-instance attribute exposing the torch.distributed world."""

    def __init__(self, what):
        self.what = what

    def __get__(self, obj, owner=None):
        from ..parallel import process_group as pgm

        if self.what == "comm":
            return pgm.world_group()
        if self.what == "rank":
            return pgm.world_rank()
        return pgm.world_size()


class _ParallelMixin:
    """Collective fit: every rank calls ``fit`` and every rank gets the full tree.

    Reference contract (``mpitree/tree/decision_tree.py:310-362``): each rank
    passes the same full ``X, y``. ``strategy`` selects how the work is split
    across ranks (see :mod:`mpitree_amd.parallel.strategies`):

    * ``"feature"`` -- feature-parallel split search, one small all-gather of
      per-node candidates per level (rows replicated, as in the reference);
    * ``"data"`` -- row-sharded histograms; per level each feature block's
      histograms are reduced to the block's owner rank (a reduce-scatter by
      feature) and one all-gather of split records picks the splits;
    * ``"subtree"`` -- load-balanced subtree task parallelism (the reference's
      strategy, without its parity-split load imbalance): replicated levels
      until a level holds >= 4 units per rank, an LPT assignment of those
      units, no per-level collective, one all-gather of finished subtrees;
    * ``"auto"`` -- replicated rows: ``"subtree"`` on the GPU device loop,
      feature-parallel exact thresholds on continuous features; row-sharded
      input (``data_sharded=True``): ``"data"``.

    The process group is created lazily on first use (``nccl``/RCCL for GPU
    fits, ``gloo`` otherwise); importing the module has no side effects.
    """

    WORLD_COMM = _WorldAttr("comm")
    WORLD_RANK = _WorldAttr("rank")
    WORLD_SIZE = _WorldAttr("size")

    def fit(self, X, y, *, data_sharded: bool = False, checkpoint=None):
        """Collective fit. Failure handling the reference lacks (an exception
        on one rank there deadlocks the others, ``decision_tree.py:446-477``):
        every rank reports its status in one all-reduce after the fit, so an
        error on any rank raises on all of them; a cross-rank digest check
        (``MPITREE_CHECK_CONSISTENCY``, default on) verifies every rank holds
        the same tree. Hangs are bounded by the process-group timeout
        (``MPITREE_DIST_TIMEOUT`` seconds). ``checkpoint``: a path every rank
        passes; GPU ranks save per-rank device-loop state there after every
        level and resume from the newest level all of them hold."""
        from ..parallel.strategies import make_comm
        from ..utils.observability import maybe_inject_fault, tree_digest

        from ..parallel.failure import ABORT, CollectiveFitAborted, FitGuard

        comm, X, y = make_comm(
            getattr(self, "strategy", "auto"),
            X,
            y,
            device=self.device,
            data_sharded=data_sharded,
            regression=self._regression,
        )
        kw = dict(comm.fit_kwargs())
        if checkpoint is not None:
            kw["checkpoint"] = checkpoint
        if getattr(comm, "world_size", 1) == 1:
            return self._fit_impl(X, y, comm=comm, **kw)
        # pre-flight (fault injection / MPITREE_PREFLIGHT=1): a rank that cannot
        # start makes every rank raise instead of leaving the others blocked in a
        # collective. Off by default: every rank validates the same replicated
        # input identically, and the check costs a host-synchronising all-reduce
        error = None
        if os.environ.get("MPITREE_FAULT_RANK") or os.environ.get("MPITREE_PREFLIGHT") == "1":
            try:
                maybe_inject_fault(comm.rank)
            except Exception as e:
                error = e
            self._raise_if_any_failed(comm, error)
        # failure containment (parallel/failure.py): a rank that fails mid-fit
        # publishes it through the c10d store; peers' host loops notice and fail
        # too, or, when a peer is stuck inside a collective, the group is aborted
        # -- no rank waits for the process-group timeout
        with FitGuard(comm) as guard:
            try:
                self._fit_impl(X, y, comm=comm, **kw)
            except Exception as e:  # reported to every rank below
                error = e
                own = isinstance(e, _OWN_ERRORS)  # raised by this rank's own logic
                if isinstance(e, CollectiveFitAborted) or (ABORT.is_set() and not own):
                    # (a peer failed first: its error, not this rank's broken collective)
                    error = CollectiveFitAborted(f"collective fit aborted ({guard.describe()})")
                torn = guard.fail(error)
                if torn is not None:
                    raise torn
            # one all-gather of {failed, tree digest}: failure propagation + consistency
            # (a tree assembled in one node-shared buffer is the same memory on
            # every rank: nothing to compare)
            check = os.environ.get("MPITREE_CHECK_CONSISTENCY", "1") != "0"
            shared = (getattr(self, "fit_stats_", None) or {}).get("assembly") == "shared-host"
            digest = tree_digest(self._arrays) if (error is None and check and not shared) else 0
            try:
                st = comm._all_gather(np.array([1 if error is not None else 0, digest],
                                               np.int64))
            except Exception as e:  # a failed peer tore the group down meanwhile
                raise CollectiveFitAborted(f"collective fit aborted ({guard.describe()})") from e
        if st[:, 0].any():
            self._raise_if_any_failed(comm, error, known_failed=True)
        if check and not (st[:, 1] == st[0, 1]).all():
            raise RuntimeError("ranks built different trees (digest mismatch)")
        return self


    @staticmethod
    def _raise_if_any_failed(comm, error, known_failed=False):
        from ..utils.observability import logger

        if error is not None:
            logger.error("rank %d: collective fit failed: %r", comm.rank, error)
        if known_failed or comm.any_failed(error is not None):
            if error is not None:
                raise error
            raise RuntimeError("collective fit failed on another rank")


class ParallelDecisionTreeClassifier(_ParallelMixin, DecisionTreeClassifier):
    """Distributed decision tree classifier (collective ``fit``)."""

    def __init__(
        self,
        *,
        max_depth: int | None = None,
        min_samples_split: int = 2,
        criterion: str = "entropy",
        min_samples_leaf: int = 1,
        max_bins: int | None = None,
        device: str = "auto",
        strategy: str = "auto",
    ):
        super().__init__(
            max_depth=max_depth,
            min_samples_split=min_samples_split,
            criterion=criterion,
            min_samples_leaf=min_samples_leaf,
            max_bins=max_bins,
            device=device,
        )
        self.strategy = strategy


class ParallelDecisionTreeRegressor(_ParallelMixin, DecisionTreeRegressor):
    """Distributed regression tree (collective ``fit``)."""

    def __init__(
        self,
        *,
        max_depth: int | None = None,
        min_samples_split: int = 2,
        criterion: str = "squared_error",
        min_samples_leaf: int = 1,
        max_bins: int | None = None,
        device: str = "auto",
        strategy: str = "auto",
    ):
        super().__init__(
            max_depth=max_depth,
            min_samples_split=min_samples_split,
            criterion=criterion,
            min_samples_leaf=min_samples_leaf,
            max_bins=max_bins,
            device=device,
        )
        self.strategy = strategy


for _cls in (DecisionTreeClassifier, ParallelDecisionTreeClassifier):
    _cls.__module__ = "mpitree.tree.decision_tree"
