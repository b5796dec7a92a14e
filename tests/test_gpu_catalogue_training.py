"""The catalogue operators where the framework calls them: the trainers' softmax loss, Muon steps, evals from
8-bit scores, and a run of them together."""
import ctypes
import io

import numpy as np
import pytest
import torch

from igr import _lib as L
from igr import model as M
from igr import ops
from igr import trainer as T
from igr.optim import Adam, Muon

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda')


class DS:
    def __init__(self, nu=300, ni=200, ne=10 * 256 + 77, seed=11):
        rng = np.random.default_rng(seed)
        self.name, self.n_users, self.n_items, self.ne = 'toy', nu, ni, ne
        self.train_pairs = np.stack([rng.integers(0, nu, ne), rng.integers(0, ni, ne)], 1)
        self.train_array = self.train_pairs.tolist()
        self.train_data = [sorted(set(self.train_pairs[self.train_pairs[:, 0] == u, 1].tolist())) for u in range(nu)]
        self.val_data = [[int(rng.integers(0, ni))] for _ in range(nu)]
        self.test_data = [[int(rng.integers(0, ni))] for _ in range(nu)]

    def __len__(self):
        return self.ne


MODELS = ['LightGCN', 'NGCF', 'IGCN', 'AttIGCN', 'IMF', 'IMCGAE']


def toy(name, d=32, ds=None, **kw):
    ds = ds or DS()
    torch.manual_seed(5)
    m = M.get_model({'name': name, 'embedding_size': d, 'n_layers': 0 if name == 'IMF' else 2, 'device': DEV,
                     'dropout': 0. if name in ('NGCF', 'IMCGAE') else 0.3, 'layer_sizes': [d, d], 'feature_ratio': 1.,
                     'dataset': ds}, ds)
    igcn = name in ('IGCN', 'AttIGCN', 'IMF')
    cfg = {'name': 'IGCNTrainer' if igcn else 'BPRTrainer', 'optimizer': 'Adam', 'lr': 1e-2, 'l2_reg': 1e-4,
           'aux_reg': 0.01, 'device': DEV, 'n_epochs': 2, 'batch_size': 256, 'test_batch_size': 512,
           'topks': [1, 5, 10, 15, 20], 'seed': 3, 'graph': False, 'loss': 'softmax', 'temperature': 0.5}
    cfg.update(kw)
    return m, T.get_trainer(cfg, ds, m)


def params(m):
    torch.cuda.synchronize()
    return {k: v.detach().clone() for k, v in m.state_dict().items() if v.dtype == torch.float32}


@pytest.mark.parametrize('name', MODELS)
def test_model_softmax_loss_against_the_formula(name):
    """Loss and l2 from the model's own rep in 64 bits; the table's gradient as the formula's gradient of
    rep sent back through the same propagation.  The loss operator is off by a few 2^-20 of a
    row's gradient and the propagation's own fp32 sums add as much, on both sides: 1e-4 of the
    gradient's largest entry holds them apart from any mistake of a term."""
    m, _ = toy(name)
    m.eval()
    u = torch.randint(0, 300, (256,), device=DEV)
    p = torch.randint(0, 200, (256,), device=DEV)
    loss, l2 = m.softmax_loss(u, p, scale=2.0)
    (loss + 0.1 * l2).backward()
    got = {k: v.grad.clone() for k, v in m.named_parameters() if v.grad is not None}
    m.zero_grad()
    rep = m.get_rep()
    r = rep.detach().double().requires_grad_()
    ref = torch.nn.functional.cross_entropy(2.0 * r[u].matmul(r[300:].t()), p)
    e = m.embedding.weight.detach().double().requires_grad_() if name == 'LightGCN' else r
    ref_l2 = (e[u].square().sum(1) + e[300 + p].square().sum(1)).mean()
    if name == 'AttIGCN':
        extra = m.weight_q.weight.square().sum() + m.weight_k.weight.square().sum()
        (0.1 * extra).backward()
        ref_l2 = ref_l2 + float(extra.detach())
    (ref + 0.1 * ref_l2).backward()
    assert abs(float(loss.detach()) - float(ref.detach())) < 1e-5 * float(ref.detach())
    assert abs(float(l2.detach()) - float(ref_l2.detach())) < 1e-5 * float(ref_l2.detach())
    rep.backward(r.grad.float())
    if name == 'LightGCN':
        m.embedding.weight.grad.add_(e.grad.float())
    for k, v in m.named_parameters():
        if k in got:
            assert (got[k] - v.grad).abs().max() <= 1e-4 * v.grad.abs().max() + 1e-9, k
    assert m.softmax_loss(u, p, need_l2=False)[1] is None


@pytest.mark.parametrize('name', MODELS)
@pytest.mark.parametrize('optimizer', ['Adam', 'Muon'])
def test_captured_softmax_epochs_match_eager_epochs(name, optimizer):
    me, te = toy(name, optimizer=optimizer)
    mg, tg = toy(name, optimizer=optimizer, graph=True)
    for epoch in range(2):
        me.train()
        mg.train()
        le, pe = te.train_one_epoch(), params(me)
        lg, pg = tg.train_one_epoch(), params(mg)
        assert le == lg, (epoch, le, lg)
        for k in pe:
            assert torch.equal(pg[k], pe[k]), (epoch, k)
    tg._close_step_graph()


def test_bpr_stays_the_default():
    _, tr = toy('LightGCN')
    assert tr.loss == 'softmax'
    ds = DS()
    m, _ = toy('LightGCN', ds=ds)
    cfg = {k: v for k, v in tr.config.items() if k not in ('loss', 'temperature')}
    t = T.get_trainer(cfg, ds, m)
    assert t.loss == 'bpr' and t.score_dtype == 'float32' and type(t.opt) is Adam


def test_trainer_refusals():
    for kw, msg in ((dict(loss='hinge'), 'loss'), (dict(temperature=0.0), 'temperature'),
                    (dict(temperature=float('nan')), 'temperature'), (dict(fused=False), 'unfused'),
                    (dict(score_dtype='int4'), 'score_dtype')):
        with pytest.raises(ValueError, match=msg):
            toy('LightGCN', **kw)
    m, tr = toy('LightGCN', d=300)
    with pytest.raises(L.IgrError, match='width'):
        tr.step(*[torch.zeros(4, dtype=torch.int64, device=DEV)] * 3)


def test_int8_ranking_equals_the_float_ranking_of_whole_numbers():
    """Rows of whole numbers whose largest is 127 are their own 8-bit rows (up to one scale a row, here 1), and
    their products are exact in both forms: the same ranking, ties included."""
    ds = DS()
    m, tr = toy('LightGCN', ds=ds)
    m.eval()
    gen = torch.Generator(device=DEV).manual_seed(1)
    rep = torch.randint(-126, 127, (500, 32), device=DEV, generator=gen).float()
    rep[:, 5] = 127.0
    m.get_rep = lambda: rep
    ref = {s: tr.rank(s) for s in ('train', 'val', 'test')}
    tr8 = T.get_trainer(dict(tr.config, score_dtype='int8'), ds, m)
    for s in ref:
        assert np.array_equal(ref[s], tr8.rank(s)), s
        banned = np.arange(0, 200, 3)
        assert np.array_equal(tr.rank(s, banned), tr8.rank(s, banned)), s


def test_int8_eval_ranks_the_8_bit_scores():
    ds = DS()
    m, tr = toy('IGCN', ds=ds, score_dtype='int8')
    m.eval()
    with torch.no_grad():
        rep = m.get_rep()
        q, s = ops.quantize_rows(rep)
        scores = ops.gemm_int8(q[:300], s[:300], q[300:], s[300:])
    for u in range(300):
        scores[u, ds.train_data[u]] = -np.inf
    order = scores.cpu().numpy()
    rec = tr.rank('val')
    for u in range(300):
        assert np.array_equal(rec[u], np.lexsort((np.arange(200), -order[u]))[:20]), u
    res, metrics, _ = tr.eval('test')
    assert 0.0 <= metrics['Recall'][20] <= 1.0 and 'Recall' in res


def ns64(g, steps=5, coeffs=ops.NEWTON_SCHULZ_COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = g / (g.square().sum().sqrt() + eps)
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    for _ in range(steps):
        y = x.matmul(x.t())
        x = a * x + (b * y + c * y.matmul(y)).matmul(x)
    return x.t() if flip else x


@pytest.mark.parametrize('nesterov,wd', [(True, 0.0), (False, 0.1)])
def test_muon_against_the_rule_in_64_bits(nesterov, wd):
    """Three steps of weights of several shapes (more than one launch of a shape among them).  A step is off by
    lr times the orthogonalised direction's error, 2e-4 of its norm at most (its own test), and fp32
    roundings of the parameter."""
    torch.manual_seed(0)
    shapes = [(64, 64)] * 18 + [(256, 64), (64, 256), (1, 7), (130, 300), (5, 3)]
    ps = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in shapes]
    bias = torch.nn.Parameter(torch.randn(64, device=DEV))
    opt = Muon([{'params': ps, 'orthogonal': True, 'weight_decay': wd}, {'params': [bias]}], lr=1e-2, orthogonal_lr=0.05,
               momentum=0.9, nesterov=nesterov)
    twin = torch.nn.Parameter(bias.detach().clone())
    adam = Adam([twin], lr=1e-2)
    ref = [p.detach().double().clone() for p in ps]
    mom = [torch.zeros_like(r) for r in ref]
    for _ in range(3):
        for p in ps + [bias]:
            p.grad = torch.randn_like(p) * 0.1
        twin.grad = bias.grad.clone()
        opt.step()
        adam.step()
        for i, p in enumerate(ps):
            g = p.grad.double()
            mom[i] = 0.9 * mom[i] + g
            u = ns64(g + 0.9 * mom[i] if nesterov else mom[i])
            ref[i] = (1 - 0.05 * wd) * ref[i] - 0.05 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * u
    assert torch.equal(bias, twin)  # the other group is Adam's, bit for bit
    for i, p in enumerate(ps):
        lr = 0.05 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        err = (p.detach().double() - ref[i]).square().sum().sqrt()
        norm = min(p.shape) ** 0.5
        assert err <= 3 * lr * 2e-4 * 1.2 * norm + 12 * 2.0 ** -24 * ref[i].square().sum().sqrt(), (p.shape, float(err))


def test_muon_takes_the_dense_layers_of_a_model():
    m, tr = toy('NGCF', optimizer='Muon', orthogonal_lr=0.03)
    assert isinstance(tr.opt, Muon)
    groups = {g['orthogonal']: g for g in tr.opt.param_groups}
    dense = {id(x.weight) for x in list(m.gc_layers) + list(m.bi_layers)}
    assert {id(p) for p in groups[True]['params']} == dense and groups[True]['lr'] == 0.03
    assert {id(p) for p in groups[False]['params']} == {id(p) for p in m.parameters()} - dense
    assert groups[False]['lr'] == 1e-2
    m, tr = toy('LightGCN', optimizer='Muon')  # no dense layers: Adam for all
    assert [g['orthogonal'] for g in tr.opt.param_groups] == [False]
    plain = Muon([torch.nn.Parameter(torch.zeros(3, 4, device=DEV)), torch.nn.Parameter(torch.zeros(4, device=DEV))])
    assert [g['orthogonal'] for g in plain.param_groups] == [True, False]
    with pytest.raises(ValueError, match='2-D'):
        Muon([{'params': [torch.nn.Parameter(torch.zeros(4, device=DEV))], 'orthogonal': True}])
    with pytest.raises(ValueError, match='hyper'):
        Muon([torch.nn.Parameter(torch.zeros(3, 4, device=DEV))], momentum=1.0)


def test_muon_state_survives_a_checkpoint():
    torch.manual_seed(1)
    p = torch.nn.Parameter(torch.randn(64, 64, device=DEV))
    opt = Muon([p])
    gs = [torch.randn(64, 64, device=DEV) for _ in range(4)]
    for g in gs[:2]:
        p.grad = g
        opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    other = Muon([q])
    buf = io.BytesIO()  # through a file: loaded in place, the two would share their buffers
    torch.save(opt.state_dict(), buf)
    buf.seek(0)
    other.load_state_dict(torch.load(buf, weights_only=True))
    for g in gs[2:]:
        p.grad, q.grad = g, g.clone()
        opt.step()
        other.step()
    assert torch.equal(p, q)


def test_muon_leaves_parameters_without_gradients_alone():
    p, q = (torch.nn.Parameter(torch.randn(8, 8, device=DEV)) for _ in range(2))
    opt = Muon([p, q])
    before = q.detach().clone()
    p.grad = torch.randn(8, 8, device=DEV).t()  # not contiguous
    opt.step()
    assert torch.equal(q, before) and not opt.state.get(q)


def test_train_rank_and_reload_together(tmp_path):
    """Softmax loss, Muon and 8-bit evals through train(): the epochs run captured, evals rank, the best
    checkpoint comes back."""
    m, tr = toy('NGCF', d=64, optimizer='Muon', score_dtype='int8', graph='auto', checkpoint_dir=str(tmp_path))
    best = tr.train(verbose=False)
    assert np.isfinite(best) and tr.save_path is not None
    assert getattr(tr, '_step_graph', None) is None
    for v in m.state_dict().values():
        assert torch.isfinite(v).all()


def test_muon_c_arguments_on_the_device():
    p = torch.zeros(8, device=DEV)
    s = (L.IgrMuonSlot * 1)()
    s[0].direction, s[0].n = p.data_ptr(), 8
    f = L.lib().igr_muon_direction_f32
    assert f(1, ctypes.addressof(s), 0.9, 1, None) == 1 and b'NULL' in L.lib().igr_last_error()
