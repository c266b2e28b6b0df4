#!/usr/bin/env python
"""The reference's Keras flavour (``HorovodKeras/src/imagenet_keras_horovod.py``) on this
framework: weight decay 5e-5 on kernels, LR warm-up (5 epochs) + step schedule (x0.1 @30,
x0.01 @60, x0.001 @80), metric averaging, broadcast at start, rank-0 checkpoints with working
resume (the reference hard-codes ``resume_from_epoch = 0``), optional validation allreduce.
"""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import distributeddeeplearning_amd.torch as hvd  # noqa: E402
from distributeddeeplearning_amd import callbacks as cb  # noqa: E402
from distributeddeeplearning_amd.models import build_model  # noqa: E402
from distributeddeeplearning_amd.optim import FusedLARS, FusedMuon, FusedSGD  # noqa: E402
from distributeddeeplearning_amd.training import Trainer, build_data  # noqa: E402
from distributeddeeplearning_amd.utils import TrainConfig, get_logger  # noqa: E402
from distributeddeeplearning_amd.utils import checkpoint  # noqa: E402


def get_hooks(cfg, logger, data_length, model_dir, is_distributed, verbose):
    """Reference ``_get_hooks`` (:194-227)."""
    hooks = []
    if is_distributed:
        hooks += [cb.BroadcastGlobalVariablesCallback(0), cb.MetricAverageCallback()]
        hooks += cb.default_imagenet_schedule(warmup_epochs=cfg.warmup_epochs or 5, verbose=verbose)
    hooks.append(cb.LoggerCallback(logger, data_length))
    if model_dir and (not is_distributed or hvd.rank() == 0):
        hooks.append(cb.CheckpointCallback(model_dir))
    return hooks


def main(argv=None):
    cfg = TrainConfig.from_args(argv)
    if cfg.weight_decay == 0.0:
        cfg.weight_decay = 5e-5  # reference _WEIGHT_DECAY (:42), applied as L2 on kernels (:104-109)
    logger = get_logger()
    hvd.init()
    use_cuda = torch.cuda.is_available()
    world, rank = hvd.size(), hvd.rank()
    device = torch.device("cuda", torch.cuda.current_device()) if use_cuda else torch.device("cpu")
    dtype = torch.bfloat16 if (cfg.dtype == "bf16" and use_cuda) else torch.float32
    verbose = 1 if rank == 0 else 0

    # resume_from_epoch is decided on rank 0 and broadcast (:287-291)
    resume_from_epoch = checkpoint.latest_epoch(cfg.output_dir) if (rank == 0 and cfg.output_dir) else 0
    resume_from_epoch = hvd.broadcast(resume_from_epoch, 0, name="resume_from_epoch")

    train_loader, val_loader, data_length, _ = build_data(cfg, device, dtype, logger, world, rank)
    model = build_model(cfg.model, num_classes=cfg.num_classes)
    model.to_compute(device, dtype) if dtype == torch.bfloat16 else model.to(device)
    opt_cls = {"lars": FusedLARS, "muon": FusedMuon}.get(cfg.optimizer, FusedSGD)
    opt = opt_cls(model.named_parameters(), lr=cfg.lr * world, momentum=cfg.momentum,
                  weight_decay=cfg.weight_decay)
    opt = hvd.DistributedOptimizer(opt, named_parameters=model.named_parameters())
    if resume_from_epoch > 0 and cfg.output_dir:
        checkpoint.resume(cfg.output_dir, model, opt)

    model_dir = checkpoint.model_dir(cfg.output_dir, cfg.temp_dir)
    trainer = Trainer(model, opt, callbacks=get_hooks(cfg, logger, data_length, model_dir,
                                                      world > 1 or cfg.distributed, verbose))
    steps = len(train_loader) if not cfg.max_steps else min(len(train_loader), cfg.max_steps)
    logger.info("Training ...")
    trainer.fit(train_loader, epochs=cfg.epochs, initial_epoch=resume_from_epoch,
                steps_per_epoch=steps, verbose=verbose)
    if cfg.validation and val_loader is not None:
        score = trainer.evaluate(val_loader)
        if verbose:
            print("Test loss:", score[0])
            print("Test accuracy:", score[1])
    hvd.shutdown()


if __name__ == "__main__":
    main()
