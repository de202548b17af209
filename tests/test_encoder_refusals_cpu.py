"""CPU: encoders that carry BERT's names but compute something else are refused when the packed encoder is built."""
import pytest
import torch
from torch import nn

transformers = pytest.importorskip("transformers")

SIZES = dict(vocab_size=50, hidden_size=32, num_hidden_layers=2, num_attention_heads=2, intermediate_size=64, max_position_embeddings=40)


def build(model):
    from two_towers_overlords_amd.encoder import PackedBertEncoder

    return PackedBertEncoder(model)


def test_a_bert_is_taken():
    assert build(transformers.BertModel(transformers.BertConfig(**SIZES))).heads == 2


@pytest.mark.parametrize("family", ["Roberta", "XLMRoberta", "Camembert", "Electra", "Ernie"])
def test_other_families_are_refused(family):
    """RoBERTa's positions start behind the padding id and skip padded tokens; ELECTRA projects its embeddings; ERNIE adds task
    embeddings: each has every submodule that a BERT has."""
    model = getattr(transformers, f"{family}Model")(getattr(transformers, f"{family}Config")(**SIZES))
    with pytest.raises(ValueError, match="BERT-shaped"):
        build(model)


def test_layers_whose_weight_is_not_all_of_them_are_refused():
    class Adapted(nn.Linear):
        def __init__(self, of):
            super().__init__(of.in_features, of.out_features)
            self.down, self.up = nn.Linear(of.in_features, 2, bias=False), nn.Linear(2, of.out_features, bias=False)

        def forward(self, x):
            return super().forward(x) + self.up(self.down(x))

    for swap in (lambda l: setattr(l.attention.self, "query", Adapted(l.attention.self.query)),
                 lambda l: setattr(l.output, "dense", Adapted(l.output.dense)),
                 lambda l: setattr(l.output, "LayerNorm", nn.Identity())):
        model = transformers.BertModel(transformers.BertConfig(**SIZES))
        swap(model.encoder.layer[1])
        with pytest.raises(ValueError, match="plain layers"):
            build(model)


def test_a_parametrised_weight_is_still_read():
    model = transformers.BertModel(transformers.BertConfig(**SIZES))
    nn.utils.parametrizations.orthogonal(model.encoder.layer[0].attention.self.query)
    build(model)
    assert isinstance(model.encoder.layer[0].attention.self.query.weight, torch.Tensor)
