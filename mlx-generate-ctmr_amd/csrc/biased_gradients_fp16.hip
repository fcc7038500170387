#include "biased_gradients.hpp"

CTMR_BIASED_GRADIENTS(_Float16)
