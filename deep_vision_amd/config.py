"""Typed training-configuration registry.

Every entry reproduces one reference configuration exactly (batch, optimizer and its
parameters, scheduler, epochs, workers, model kwargs) with its source cited. The PyTorch
classifier configs (R/ResNet/pytorch/train.py:26-215, R/LeNet/pytorch/train.py:15-32) use a
**global** batch that the data-parallel launcher splits across ranks; the TF2-origin configs
(YOLO / Hourglass / CenterNet, MirroredStrategy) use a **per-replica** batch x world.

Differences from the reference, all additive or documented fixes:
  * ``resnet152`` is registered with the resnet50 hyper-parameters;
  * ``shufflenet1`` (reference file empty, A-M9d) uses the MobileNet recipe;
  * the TF1-Keras ``kernel_regularizer=l2(1e-4)`` becomes SGD weight decay 2e-4
    (d/dw of 1e-4 * w^2).
"""
from __future__ import annotations

import copy
import dataclasses
from dataclasses import dataclass, field
from typing import Any, Dict, Optional, Tuple


@dataclass
class TrainConfig:
    name: str
    model: str                      # deep_vision_amd.models.MODELS key
    batch_size: int                 # global (batch_semantics == "global") or per replica
    total_epochs: int
    optimizer: str                  # "sgd" | "adam" | "adamw" | "rmsprop"
    optimizer_params: Dict[str, Any]
    scheduler: Optional[str] = None  # "plateau" | "step" | "lambda" | "manual_plateau" | "linear_decay" | None
    scheduler_params: Dict[str, Any] = field(default_factory=dict)
    num_workers: int = 4
    model_params: Dict[str, Any] = field(default_factory=dict)
    family: str = "classification"  # classification | yolo | hourglass | centernet | dcgan | cyclegan
    dataset: str = "imagenet"       # imagenet | mnist | coco | mpii | cyclegan | synthetic
    input_shape: Tuple[int, int, int] = (3, 224, 224)
    batch_semantics: str = "global"
    checkpoint_dir: str = "./saved_models/"
    source: str = ""                # reference file:lines of the original entry
    extras: Dict[str, Any] = field(default_factory=dict)

    def replace(self, **kw) -> "TrainConfig":
        return dataclasses.replace(copy.deepcopy(self), **kw)

    def per_rank_batch(self, world: int) -> int:
        if self.batch_semantics == "per_replica":
            return self.batch_size
        if self.batch_size % world:
            raise ValueError(f"global batch {self.batch_size} is not divisible by world size {world}")
        return self.batch_size // world

    def global_batch(self, world: int) -> int:
        return self.batch_size * world if self.batch_semantics == "per_replica" else self.batch_size

    def get(self, key, default=None):  # dict-style access used by the reference's run_epochs
        return getattr(self, key, self.extras.get(key, default))


def _sgd(lr, wd, momentum=0.9):
    return {"lr": lr, "momentum": momentum, "weight_decay": wd}


_PLATEAU = ("plateau", {"mode": "max", "factor": 0.1})
_IMAGENET = dict(dataset="imagenet", input_shape=(3, 224, 224))

CONFIGS: Dict[str, TrainConfig] = {}


def register(cfg: TrainConfig) -> TrainConfig:
    CONFIGS[cfg.name] = cfg
    return cfg


# ---------------- PyTorch classifiers (R/ResNet/pytorch/train.py:26-215) ----------------
register(TrainConfig("lenet5", "lenet5", 64, 50, "adam", {"lr": 1e-3}, *_PLATEAU, num_workers=2,
                     dataset="mnist", input_shape=(1, 32, 32), source="R/LeNet/pytorch/train.py:15-32"))
register(TrainConfig("alexnet1", "alexnet1", 128, 200, "sgd", _sgd(0.01, 5e-4), *_PLATEAU, num_workers=1, **_IMAGENET,
                     source="R/ResNet/pytorch/train.py:27-51"))
register(TrainConfig("alexnet2", "alexnet2", 128, 200, "sgd", _sgd(0.01, 5e-4), *_PLATEAU, num_workers=16, **_IMAGENET,
                     source="R/ResNet/pytorch/train.py:52-74"))
register(TrainConfig("vgg16", "vgg16", 128, 200, "sgd", _sgd(0.01, 5e-4), "step", {"step_size": 10, "gamma": 0.5},
                     num_workers=16, **_IMAGENET, source="R/ResNet/pytorch/train.py:75-99"))
register(TrainConfig("vgg19", "vgg19", 64, 200, "sgd", _sgd(0.01, 5e-4), "step", {"step_size": 10, "gamma": 0.5},
                     num_workers=16, **_IMAGENET, source="R/ResNet/pytorch/train.py:100-118"))
register(TrainConfig("inception1", "inception1", 128, 200, "sgd", _sgd(0.01, 2e-4), "lambda",
                     {"lr_lambda": "inception_poly"}, num_workers=16, **_IMAGENET,
                     extras={"aux_weight": 0.3}, source="R/ResNet/pytorch/train.py:119-140"))
register(TrainConfig("resnet34", "resnet34", 256, 200, "sgd", _sgd(0.1, 1e-4), *_PLATEAU, num_workers=16, **_IMAGENET,
                     source="R/ResNet/pytorch/train.py:141-165"))
register(TrainConfig("resnet50", "resnet50", 256, 200, "sgd", _sgd(0.1, 1e-4), *_PLATEAU, num_workers=16, **_IMAGENET,
                     source="R/ResNet/pytorch/train.py:166-184"))
register(TrainConfig("resnet152", "resnet152", 256, 200, "sgd", _sgd(0.1, 1e-4), *_PLATEAU, num_workers=16, **_IMAGENET,
                     source="SURVEY A6 (resnet50 recipe)"))
register(TrainConfig("mobilenet1", "mobilenet1", 128, 200, "rmsprop", {"lr": 0.045, "alpha": 0.9, "eps": 1.0}, "step",
                     {"step_size": 2, "gamma": 0.94}, num_workers=16, model_params={"alpha": 1}, **_IMAGENET,
                     source="R/ResNet/pytorch/train.py:185-214"))
register(TrainConfig("shufflenet1", "shufflenet1", 128, 200, "rmsprop", {"lr": 0.045, "alpha": 0.9, "eps": 1.0}, "step",
                     {"step_size": 2, "gamma": 0.94}, num_workers=16, **_IMAGENET,
                     source="reference file empty; MobileNet recipe"))

# ---------------- TF1-Keras classifiers (R/ResNet/tensorflow/train.py:21-62) ----------------
_KERAS_PLATEAU = ("plateau", {"mode": "min", "factor": 0.1, "patience": 10, "min_lr": 1e-5, "metric": "val_loss"})
register(TrainConfig("alexnet2_tf", "alexnet2_tf", 128, 200, "sgd", _sgd(0.01, 0.0), *_KERAS_PLATEAU, **_IMAGENET,
                     extras={"gpus": 1, "keras": True}, source="R/ResNet/tensorflow/train.py:22-35"))
register(TrainConfig("resnet50_tf", "resnet50_tf", 128, 200, "sgd", _sgd(0.01, 2e-4), *_KERAS_PLATEAU, **_IMAGENET,
                     extras={"keras": True}, source="R/ResNet/tensorflow/train.py:36-48"))
register(TrainConfig("resnet152_tf", "resnet152_tf", 128, 200, "sgd", _sgd(0.01, 2e-4), *_KERAS_PLATEAU, **_IMAGENET,
                     extras={"keras": True}, source="R/ResNet/tensorflow/train.py:49-61"))
register(TrainConfig("lenet5_tf", "lenet5_tf", 64, 50, "adam", {"lr": 1e-3}, None, {}, dataset="mnist",
                     input_shape=(1, 32, 32), extras={"keras": True, "scale_only": True},
                     source="R/LeNet/tensorflow/train.py:13-24"))
register(TrainConfig("mobilenet1_tf", "mobilenet1_tf", 32, 10, "rmsprop", {"lr": 0.045, "alpha": 0.9, "eps": 1.0},
                     "step", {"step_size": 2, "gamma": 0.94}, **_IMAGENET, batch_semantics="per_replica",
                     extras={"keras": True}, source="R/MobileNet/tensorflow/train.py:7-14 (skeleton: optimizer undefined there, PT recipe used)"))

# ---------------- TF2 custom-loop families (MirroredStrategy: per-replica batch) ----------------
register(TrainConfig("yolov3", "yolov3", 16, 300, "adam", {"lr": 0.01}, "manual_plateau",
                     {"factor": 0.1, "max_patience": 10}, family="yolo", dataset="coco", input_shape=(3, 416, 416),
                     model_params={"num_classes": 80}, batch_semantics="per_replica", checkpoint_dir="./models/",
                     extras={"version": "1.0.1", "seed": 1}, source="R/YOLO/tensorflow/train.py:13-19,46-68"))
register(TrainConfig("hourglass", "hourglass104", 32, 100, "adam", {"lr": 1e-3}, "manual_plateau",
                     {"factor": 0.1, "max_patience": 10, "inclusive": True}, family="hourglass", dataset="mpii", input_shape=(3, 256, 256),
                     model_params={"num_stack": 4, "num_residual": 1, "num_heatmap": 16},
                     batch_semantics="per_replica", checkpoint_dir="./models/",
                     extras={"version": "1.0.1", "fg_weight": 81.0}, source="R/Hourglass/tensorflow/main.py:22-33"))
register(TrainConfig("centernet", "centernet", 16, 300, "adam", {"lr": 0.01}, "manual_plateau",
                     {"factor": 0.1, "max_patience": 10}, family="centernet", dataset="coco",
                     input_shape=(3, 256, 256), model_params={"num_classes": 80, "num_stack": 2},
                     batch_semantics="per_replica", checkpoint_dir="./models/", extras={"version": "1.0.0"},
                     source="R/ObjectsAsPoints/tensorflow/train.py:13-17,35-45"))
register(TrainConfig("dcgan", "dcgan", 256, 50, "adam", {"lr": 1e-4}, None, {}, family="dcgan", dataset="mnist",
                     input_shape=(1, 28, 28), checkpoint_dir="./checkpoints/",
                     extras={"noise_dim": 100, "num_examples_to_generate": 16, "save_every": 2, "keep": 3},
                     source="R/DCGAN/tensorflow/main.py:13-17,31-32"))
register(TrainConfig("cyclegan", "cyclegan", 4, 200, "adam", {"lr": 2e-4, "betas": (0.5, 0.999)}, "linear_decay",
                     {"decay_epoch": 100}, family="cyclegan", dataset="cyclegan", input_shape=(3, 256, 256),
                     model_params={"n_blocks": 9}, checkpoint_dir="./checkpoints-{dataset}/",
                     extras={"lambda_cycle": 10.0, "lambda_identity": 5.0, "pool_size": 50, "shuffle": 10000,
                             "save_every": 2, "dataset_name": "horse2zebra"},
                     source="R/CycleGAN/tensorflow/train.py:14-21,122-131"))


def get_config(name: str, **overrides) -> TrainConfig:
    try:
        cfg = CONFIGS[name]
    except KeyError:
        raise KeyError(f"unknown config {name!r}; available: {sorted(CONFIGS)}") from None
    return cfg.replace(**overrides) if overrides else copy.deepcopy(cfg)


def inception_poly(epoch: int) -> float:
    """R/ResNet/pytorch/train.py:137: (1 - e/60)^.5 for e < 60, then .01, then .001 after 75."""
    if epoch < 60:
        return (1 - epoch / 60) ** 0.5
    return 0.01 if epoch < 75 else 0.001


LR_LAMBDAS = {"inception_poly": inception_poly}
