"""One rank of a data-parallel Muon run on CPU tensors: DistributedOptimizer(Muon) beside
DistributedOptimizer(FusedAdam), each rank with its own half of the batch."""
import json
import sys

import torch

import mihvd.torch as hvd
from mihvd.models.bert import BertConfig, BertForMaskedLM, muon_parameters, synthetic_mlm_batch
from mihvd.optim import FusedAdam, Muon


def main(out):
    hvd.init()
    torch.manual_seed(0)
    c = BertConfig(vocab_size=53, hidden=16, layers=1, heads=2, ffn=24, max_len=8, dropout=0.0, ffn_impl="swiglu",
                   loss_impl="fused")
    model = BertForMaskedLM(c)
    hvd.broadcast_parameters(model.state_dict(), root_rank=0)
    matrices, others = muon_parameters(model)

    def wrap(o):
        mine = {id(p) for g in o.param_groups for p in g["params"]}
        return hvd.DistributedOptimizer(o, named_parameters=[(k, p) for k, p in model.named_parameters() if id(p) in mine])

    opts = [wrap(Muon(matrices, lr=0.02)), wrap(FusedAdam(others, lr=1e-2))]
    g = torch.Generator().manual_seed(7)
    ids, _ = synthetic_mlm_batch(4, 8, 53, "cpu", generator=g)
    ids = ids.clamp_max(52)
    labels = ids.clone()  # every position labelled: the halves weigh the same
    lo, hi = hvd.rank() * 4 // hvd.size(), (hvd.rank() + 1) * 4 // hvd.size()
    for _ in range(3):
        for o in opts:
            o.zero_grad(set_to_none=False)
        model(ids[lo:hi], labels[lo:hi]).backward()
        for o in opts:
            o.step()
    flat = torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    with open("%s.%d.json" % (out, hvd.rank()), "w") as f:
        json.dump(flat.double().tolist(), f)
    hvd.shutdown()


if __name__ == "__main__":
    main(sys.argv[1])
