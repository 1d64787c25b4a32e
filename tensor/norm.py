"""`tensor.norm`: layer norm and dropout of a model's input rows; the implementation lives in tensornetworksfork_amd.tensor.norm."""
from tensornetworksfork_amd.tensor.norm import *  # noqa: F401,F403
from tensornetworksfork_amd.tensor import norm as _impl

globals().update({k: v for k, v in vars(_impl).items() if not k.startswith('__')})
