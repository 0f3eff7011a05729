from . import functional  # noqa: F401
from .modules import (AvgPool2d, BatchNorm2d, Conv2d, GatedLinear, Linear, MaxPool2d,  # noqa: F401
                      ReLU, Sequential)
