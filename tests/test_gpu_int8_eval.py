"""Evals from 8-bit rows go through the model's own predict."""
import numpy as np
import pytest
import torch

from igr import model as M
from igr import ops
from igr import trainer as T

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda')


class DS:
    def __init__(self, nu=90, ni=70, ne=900, seed=2):
        rng = np.random.default_rng(seed)
        self.name, self.n_users, self.n_items, self.ne = 'toy', nu, ni, ne
        self.train_pairs = np.stack([rng.integers(0, nu, ne), rng.integers(0, ni, ne)], 1)
        self.train_array = self.train_pairs.tolist()
        self.train_data = [sorted(set(self.train_pairs[self.train_pairs[:, 0] == u, 1].tolist())) for u in range(nu)]
        self.val_data = [[int(rng.integers(0, ni))] for _ in range(nu)]
        self.test_data = [[int(rng.integers(0, ni))] for _ in range(nu)]

    def __len__(self):
        return self.ne


class Biased(M.LightGCN):
    """Scores with a term of the item's own."""

    def predict(self, users, rep=None):
        return super().predict(users, rep) + self.bias


class Cosine(M.LightGCN):
    """Scores that no product of two 8-bit tables gives."""

    def predict(self, users, rep=None):
        rep = self.get_rep() if rep is None else rep
        rep = torch.nn.functional.normalize(rep, dim=1)
        return rep[users] @ rep[self.n_users:].t()


def build(cls):
    ds = DS()
    torch.manual_seed(5)
    m = cls({'name': 'LightGCN', 'embedding_size': 32, 'n_layers': 2, 'device': DEV, 'dataset': ds})
    cfg = {'name': 'BPRTrainer', 'optimizer': 'Adam', 'lr': 1e-2, 'l2_reg': 1e-4, 'device': DEV, 'n_epochs': 1, 'batch_size': 64,
           'test_batch_size': 32, 'topks': [1, 5, 10, 15, 20], 'seed': 3, 'score_dtype': 'int8'}
    return ds, m, T.get_trainer(cfg, ds, m)


def test_a_models_own_scores_are_ranked():
    ds, m, tr = build(Biased)
    m.bias = torch.randn(70, device=DEV)
    m.eval()
    with torch.no_grad():
        q, s = ops.quantize_rows(m.get_rep())
        scores = ops.gemm_int8(q[:90], s[:90], q[90:], s[90:]) + m.bias
    order = scores.cpu().numpy()
    rec = tr.rank('train')
    for u in range(90):
        assert np.array_equal(rec[u], np.lexsort((np.arange(70), -order[u]))[:20]), u


def test_a_model_that_cannot_score_from_8_bit_rows_is_not_ranked_by_others():
    _, m, tr = build(Cosine)
    with pytest.raises((TypeError, AttributeError)):
        tr.rank('train')


def test_predict_from_a_quantized_table():
    _, m, _ = build(M.LightGCN)
    m.eval()
    with torch.no_grad():
        rep = m.get_rep()
    users = torch.tensor([4, 0, 89, 4], device=DEV)
    q, s = ops.quantize_rows(rep)
    got = m.predict(users, ops.QuantizedTable(q, s))
    assert torch.equal(got, ops.gemm_int8(q[users], s[users], q[90:], s[90:]))
    # half a quantisation step for each operand (32 columns)
    eu, ew = 0.5 * s.double()[users][:, None], 0.5 * s.double()[90:][None, :]
    r = rep.double()
    bound = eu * r[90:].abs().sum(1)[None, :] + ew * r[users].abs().sum(1)[:, None] + 32 * eu * ew
    ref = r[users].matmul(r[90:].t().contiguous())
    assert ((got.double() - ref).abs() <= bound * (1 + 1e-4) + 1e-6 * ref.abs()).all()
