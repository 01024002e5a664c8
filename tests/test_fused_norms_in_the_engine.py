"""Llama-4's fused norms of heads under the engine: tensor parallelism (a rank's heads), sharded parameters with recomputed layers."""

import pytest
from test_distributed_cpu import L4, close, run

FUSED = L4 + ["+model.fused_qk_norm=true"]


@pytest.fixture(scope="module")
def single():
  return run(1, L4 + ["ici_mesh.fsdp=1"])["traj"]


@pytest.mark.parametrize("extra", [["ici_mesh.fsdp=1", "ici_mesh.tensor=2", "model/sharding=llama4-fsdp-tp"], ["ici_mesh.fsdp=2", "engine.remat_layers=all"],
                                   ["ici_mesh.fsdp=2", "engine.remat_layers=none"]], ids=["tensor", "recomputed", "saved"])
def test_fused_norms_match_the_separate_ones(single, extra):
  close(run(2, FUSED + extra)["traj"], single)


@pytest.mark.gpu
def test_recomputed_layers_on_the_kernels(cuda_lib, tmp_path):
  """The same losses and gradient norms with layers recomputed or not (a norm's gradient is added up by atomics) and, up to bf16's
  roundings, with the separate norms."""
  import torch

  from torchprime_b200.config import compose
  from torchprime_b200.data.synthetic import make_synthetic_dataset
  from torchprime_b200.models.model_utils import initialize_model_class
  from torchprime_b200.trainer import Trainer

  def steps(*extra):
    cfg = compose("default", ["model=llama-4-text-only-dummy", "model.hidden_size=512", "model.num_attention_heads=4", "model.num_key_value_heads=1",
                              "model.head_dim=128", "model.intermediate_size=256", "model.intermediate_size_mlp=512", "model.num_local_experts=4",
                              "model.vocab_size=1024", "model.num_hidden_layers=3", "model.moe_layers=[1]", "model.no_rope_layers=[1,1,0]",
                              "dataset=synthetic", "dataset.block_size=256", "task.global_batch_size=2", "task.max_steps=3", "task.optimizer.type=adamw",
                              "task.optimizer.learning_rate=1e-3", "ici_mesh.fsdp=1", "profile_start_step=-1", f"output_dir={tmp_path}", *extra])
    torch.manual_seed(0)
    model = initialize_model_class(cfg.model, device="meta")
    tr = Trainer(model=model, config=cfg, train_dataset=make_synthetic_dataset(vocab_size=1024, block_size=256, num_samples=32))
    loader = tr._get_train_dataloader()
    return [tuple(v.item() for v in tr.train_step(tr._prepare_batch(loader.next_batch()))) for _ in range(3)]

  fused = steps("+model.fused_qk_norm=true", "engine.remat_layers=none")
  recomputed = steps("+model.fused_qk_norm=true", "engine.remat_layers=all")
  separate = steps("engine.remat_layers=none")
  for (la, ga), (lb, gb), (lc, gc) in zip(fused, recomputed, separate):
    assert abs(la - lb) < 2e-3 and abs(ga - gb) < 5e-3 * max(1.0, gb), (fused, recomputed)
    assert abs(la - lc) < 0.03 and abs(ga - gc) < 0.08 * gc, (fused, separate)
