"""Options that the sharded trainer does not have are refused, not passed over (CPU)."""
import pytest

from igr.dist_train import ShardedIGCNTrainer


@pytest.mark.parametrize('key,value', [('loss', 'softmax'), ('optimizer', 'Muon'), ('score_dtype', 'int8')])
def test_options_of_the_other_trainers_are_refused(key, value):
    cfg = {'batch_size': 8, 'l2_reg': 0.0, 'aux_reg': 0.0, 'lr': 1e-3, key: value}
    with pytest.raises(ValueError, match=f'{key}.*{value}'):
        ShardedIGCNTrainer(cfg, None)


def test_the_options_it_has_pass_the_check():
    cfg = {'batch_size': 8, 'l2_reg': 0.0, 'aux_reg': 0.0, 'lr': 1e-3, 'loss': 'bpr', 'optimizer': 'Adam',
           'score_dtype': 'float32'}
    with pytest.raises(AttributeError, match='config'):  # on to the model, which is none here
        ShardedIGCNTrainer(cfg, None)
